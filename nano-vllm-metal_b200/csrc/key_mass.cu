// key_mass.cu -- accumulated attention weight of every cached key.
//
// For kv head h of sequence b, with rows (q head i of h's group, query token l) at
// positions pos = l + ctx - L:
//   mass[b, h, s] = (s < ctx - L ? mass[b, h, s] : 0) + sum_rows 2^(z[row, s] - lse[row])
// where z is the scaled score in base 2 and lse[row] = log2 sum_s 2^z[row, s] comes from
// the attention kernel that ran before on the same stream (+inf for a row without a key,
// then gives every key weight 0).  Keys of unmapped pages gain nothing.  No atomics:
// one thread (or warp) owns a key, so results do not depend on the order of anything.
//
// The denominators are known only after all keys, so the scores are needed twice.  Which way
// is cheaper depends on the rows of a kv head, M = Hq/Hkv * L:
//  * M <= 8 (decode): the attention kernel keeps its scores in the workspace, 4 M bytes a key
//    written and read once, next to the 4 D bytes of K and V that it reads anyway (M = 4,
//    D = 128: 32 bytes next to 512).  It weighs them itself when its chunks merge in a cluster
//    or not at all (paged_mma.cuh); when they merge through the workspace,
//    key_mass_scores_kernel does: the CTA that ends a long unit would hold its slot and, at the
//    end, the launch (64 requests of 2K-16K keys: 430 us, against 474 us that way; one request
//    of 1K keys 18 us on the device, against 16 us the other way).
//  * more rows (verify, chunks, prompts): 2 D bytes a key read again cost less than 8 M bytes
//    from M = D / 4 = 32 on, and prompts could not keep M x S scores at all:
//    key_mass_sm100_kernel computes them again on the tensor cores, S^T = K Q^T with the keys
//    as the 128 lanes of tensor memory, so that a thread owns a key: its sum needs no
//    exchange between threads and K enters shared memory once per 128 keys.  With 64 rows a
//    head or more the heads of a group are spread over the CTAs of a cluster, which add their
//    sums through distributed shared memory: causal rows make the first keys' CTAs the
//    longest.  Bound by the exponentials (16 a clock and SM) inside the tile loop and by the
//    start of its CTAs.
//  * everything else (fp32, other head dims): key_mass_generic_kernel.
// Measured on a B200 (32/8 heads, bf16): 64 requests of 2K-16K keys 26 us for 74 MB of scores
// (the whole scored step 430 us, 0.85 of a copy's rate for its K and V); prompts of 2 x 2048
// tokens 60 us next to 102 us of attention (570 TFLOP/s of S^T), ten of them behind its last wave.
#include <cooperative_groups.h>

#include <cstdlib>
#include <mutex>
#include <type_traits>

#include "nvm_common.cuh"
#include "nvm_internal.h"
#include "tcgen05.cuh"

namespace nvm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct MassParams {
  const void* q;
  const void* k;
  const void* ks;
  const int32_t* block_table;
  const int32_t* context_lens;
  const float* lse;
  float* mass;
  int64_t stride_b, stride_h, len;
  int q_dtype, kv_dtype, scale_dtype;
  int64_t B, Hq, Hkv, L, D, P, ps, mp, g;
  float scale_log2;
  int causal;
  int64_t window, sinks;
  int q_round;      // generic: the 16-bit type in which the attention kernel took q, or NVM_F32
  int64_t blocks;   // 1-D grids: blocks per (sequence, kv head)
};

// Any head dim <= 256, page size and dtype: a warp per key, lanes along the query rows.
constexpr int kGenWarps = 4;
__global__ void __launch_bounds__(kGenWarps * 32) key_mass_generic_kernel(MassParams p) {
  __shared__ float krow[kGenWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t bh = blockIdx.x / p.blocks, block = blockIdx.x - bh * p.blocks;
  const int64_t b = bh / p.Hkv, h = bh % p.Hkv;
  const int64_t ctx = p.context_lens[b];
  const int64_t cap = p.mp * p.ps;
  int64_t end = ctx < cap ? ctx : cap;
  if (p.len < end) end = p.len;
  for (int64_t s = block * kGenWarps + warp; s < end; s += p.blocks * kGenWarps) {
    const int64_t page = s / p.ps, off = s - page * p.ps;
    const int64_t pid = p.block_table[b * p.mp + page];
    float sum = 0.f;
    if (pid >= 0 && pid < p.P) {
      const int64_t base = (pid * p.Hkv + h) * p.ps + off;
      const float ksc = p.kv_dtype == NVM_I8 ? load_dyn(p.ks, base, p.scale_dtype) : 1.f;
      for (int64_t d = lane; d < p.D; d += 32) krow[warp][d] = load_dyn(p.k, base * p.D + d, p.kv_dtype);
      __syncwarp();
      for (int64_t r = lane; r < p.g * p.L; r += 32) {
        const int64_t l = r % p.L, pos = l + ctx - p.L;
        const bool seen = (!p.causal || s <= pos) && (p.window == 0 || s < p.sinks || s > pos - p.window);
        if (!seen) continue;
        const int64_t row = (b * p.Hq + h * p.g) * p.L + r;
        float dot = 0.f;
        for (int64_t d = 0; d < p.D; ++d) {
          float x = load_dyn(p.q, row * p.D + d, p.q_dtype);
          if (p.q_round == NVM_F16) x = __half2float(__float2half_rn(x));
          if (p.q_round == NVM_BF16) x = __bfloat162float(__float2bfloat16_rn(x));
          dot += x * krow[warp][d];
        }
        if (p.kv_dtype == NVM_I8) dot *= ksc;
        sum += exp2f(dot * p.scale_log2 - p.lse[row]);
      }
      __syncwarp();
      sum = warp_sum(sum);
    }
    if (lane == 0) {
      float* m = p.mass + b * p.stride_b + h * p.stride_h + s;
      *m = (s < ctx - p.L ? *m : 0.f) + sum;
    }
  }
}

// Scores kept by the attention kernel: [B*Hkv][v_keys][rows_pad] base-2 scores (-inf where a
// row does not see the key) on the attention kernel's virtual keys; a thread takes
// kScoreKeys keys, 256 apart, so that enough loads are in flight.
// Where the attention kernel left the units' chunks unmerged (kMerge), every CTA finds its unit's
// log-sum-exps from the chunks' (m, l), a warp a row, and one more CTA per unit merges the rows.
struct ScoreParams {
  const float* scores;
  const float2* part_ml;  // kMerge: [B*Hkv][n_chunks][rows]; else the log-sum-exps are in MassParams::lse
  const float* part_o;    // [B*Hkv][n_chunks][rows][D]
  void* out;
  int out_dtype;
  int64_t v_keys, n_chunks, ct;
  int rows;  // kRows: rows rounded up to even
};
constexpr int kScoreKeys = 4;

// kMerge: two instances, since the merge's registers cost the plain one 18 us of 430.
template <int kRows, bool kMerge>
__global__ void __launch_bounds__(256) key_mass_scores_kernel(const MassParams p, const ScoreParams sp) {
  __shared__ float s_lse[8];
  const int64_t bh = blockIdx.x / p.blocks, block = blockIdx.x - bh * p.blocks;
  const int64_t b = bh / p.Hkv, h = bh - b * p.Hkv;
  if (!kMerge && threadIdx.x < 8)
    s_lse[threadIdx.x] = (int)threadIdx.x < sp.rows ? p.lse[bh * sp.rows + threadIdx.x] : INFINITY;
  const int64_t ctx = p.context_lens[b], cap = p.mp * p.ps;
  const int64_t end = ctx < cap ? ctx : cap;
  // virtual -> real keys, as the attention kernel numbers its 16-key tiles
  int64_t tiles = (end + 15) / 16, sink_tiles = tiles, skip = 0;
  if (p.window > 0) {
    const int64_t first = ctx - p.L - p.window + 1, st = (p.sinks + 15) / 16;
    if (first > 0 && first / 16 > st && st < tiles) {
      sink_tiles = st;
      skip = first / 16 - st;
      tiles = tiles - skip > st ? tiles - skip : st;
    }
  }
  const int64_t v_end = end > 0 ? tiles * 16 : 0;
  const int64_t chunks = kMerge && end > 0 ? (tiles + sp.ct - 1) / sp.ct : 1;
  const bool merges = kMerge && block == p.blocks - 1;  // the unit's extra CTA
  if (merges ? chunks <= 1 : block * (256 * kScoreKeys) >= v_end) return;
  const int64_t part0 = bh * sp.n_chunks * sp.rows;
  if constexpr (kMerge) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float lse = INFINITY, top = -INFINITY;
    if (warp < sp.rows) {
      if (chunks <= 1) {
        lse = p.lse[bh * sp.rows + warp];
      } else {
        for (int64_t c = lane; c < chunks; c += 32) top = fmaxf(top, sp.part_ml[part0 + c * sp.rows + warp].x);
        top = warp_max(top);
        float sum = 0.f;
        for (int64_t c = lane; c < chunks; c += 32) {
          const float2 ml = sp.part_ml[part0 + c * sp.rows + warp];
          if (ml.x != -INFINITY) sum += ml.y * exp2f(ml.x - top);
        }
        sum = warp_sum(sum);
        lse = sum > 0.f ? top + log2f(sum) : INFINITY;
      }
    }
    if (lane == 0) s_lse[warp] = lse;
  }
  __syncthreads();
  if (merges) {
    // out = sum over the chunks of 2^(m - lse) O
    const int d4 = (int)p.D / 4;
    for (int i = threadIdx.x; i < sp.rows * d4; i += 256) {
      const int row = i / d4, d = (i - row * d4) * 4;
      const float lse = s_lse[row];
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int64_t c0 = 0; c0 < chunks; c0 += 8) {
        float4 v[8];
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t at = part0 + (c0 + j) * sp.rows + row;
          w[j] = c0 + j < chunks ? exp2f(sp.part_ml[at].x - lse) : 0.f;
          v[j] = c0 + j < chunks ? *reinterpret_cast<const float4*>(sp.part_o + at * p.D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (w[j] > 0.f) {  // a chunk without a key of this row holds no sum
            o.x += v[j].x * w[j];
            o.y += v[j].y * w[j];
            o.z += v[j].z * w[j];
            o.w += v[j].w * w[j];
          }
        }
      }
      const int64_t at = (bh * sp.rows + row) * p.D + d;
      store_dyn(sp.out, at, sp.out_dtype, o.x);
      store_dyn(sp.out, at + 1, sp.out_dtype, o.y);
      store_dyn(sp.out, at + 2, sp.out_dtype, o.z);
      store_dyn(sp.out, at + 3, sp.out_dtype, o.w);
    }
    return;
  }
  const int64_t v0 = block * (256 * kScoreKeys) + threadIdx.x;
  const float* z = sp.scores + bh * sp.v_keys * kRows;
  float* mrow = p.mass + b * p.stride_b + h * p.stride_h;
  float x[kScoreKeys][kRows], old[kScoreKeys];
  int64_t key[kScoreKeys];
#pragma unroll
  for (int u = 0; u < kScoreKeys; ++u) {  // every load of the thread's keys first
    const int64_t v = v0 + u * 256;
    key[u] = v >= v_end ? -1 : v / 16 >= sink_tiles ? v + skip * 16 : v;
    if (key[u] >= end || key[u] >= p.len) key[u] = -1;
    if (key[u] < 0) continue;
    old[u] = key[u] < ctx - p.L ? mrow[key[u]] : 0.f;
    if constexpr (kRows % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kRows / 4; ++i)
        *reinterpret_cast<float4*>(&x[u][4 * i]) = __ldcs(reinterpret_cast<const float4*>(z + v * kRows) + i);
    } else {
#pragma unroll
      for (int i = 0; i < kRows / 2; ++i)
        *reinterpret_cast<float2*>(&x[u][2 * i]) = __ldcs(reinterpret_cast<const float2*>(z + v * kRows) + i);
    }
  }
#pragma unroll
  for (int u = 0; u < kScoreKeys; ++u) {
    if (key[u] < 0) continue;
    float gain = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < sp.rows) gain += ex2_ftz(x[u][i] - s_lse[i]);  // an odd last column holds nothing
    mrow[key[u]] = old[u] + gain;
  }
}

// ---------------------------------------------------------------------------
// tcgen05 recomputation: a CTA per 128 keys of one (sequence, kv head)
// ---------------------------------------------------------------------------
constexpr int kMK = 128;        // keys per CTA = tensor-memory lanes
constexpr int kMR = 128;        // query rows per tile = accumulator columns
constexpr int kMThreads = 320;  // warps 0-7: exponentials; warp 8: Q copies; warp 9: MMAs
constexpr int kMCols = 256;     // two accumulators; two CTAs per SM share the 512 columns

template <int D>
struct MassSmem {
  static constexpr int kKBytes = kMK * D * 2;
  static constexpr int kQBytes = kMR * D * 2;
  static constexpr int kStages = 2;
  static constexpr int kUsed = kKBytes + kStages * kQBytes + 2 * kMR * 8 + 2 * kMK * 4 + 256;
  // at least a third of an SM's: a third CTA would only wait for tensor memory
  static constexpr int kBytes = kUsed > 80 * 1024 ? kUsed : 80 * 1024;
};

// Of 16 pairs of exponentials, the even pairs 2x with bit x set run on the FMA pipe: a quarter
// of them takes 1 % off a scored prompt (with four warps a scheduler the MUFU unit is at 80 %
// inside the tile loop).
constexpr uint32_t kPolyMask = 0x55u;

// The larger of a score and -125; NaN stays NaN.
__device__ __forceinline__ float clamp_score(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-125.f));
  return r;
}

// 2^x for a pair on the FMA pipe: n = round(x) through the 1.5 * 2^23 rounding constant,
// f = x - n in [-0.5, 0.5] (exact), a degree-5 polynomial for 2^f (near-minimax for relative
// error by iteratively reweighted least squares: 2.0e-7 in fp32, as ex2.approx), times 2^n (its
// exponent field is t's last bits; a product, since adding n to the polynomial's bits would make
// a number of a NaN).  Arguments below -125 give 2^-125 instead of a smaller number or zero, so a
// row without a key (lse = +inf) must not come here.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  constexpr float kRound = 12582912.0f;
  x.x = clamp_score(x.x);
  x.y = clamp_score(x.y);
  const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
  const float2 f = __ffma2_rn(__fadd2_rn(t, make_float2(-kRound, -kRound)), make_float2(-1.f, -1.f), x);
  float2 p = __ffma2_rn(make_float2(0.001327647f, 0.001327647f), f, make_float2(0.009675542f, 0.009675542f));
  p = __ffma2_rn(p, f, make_float2(0.055507135f, 0.055507135f));
  p = __ffma2_rn(p, f, make_float2(0.2402212f, 0.2402212f));
  p = __ffma2_rn(p, f, make_float2(0.69314694f, 0.69314694f));
  p = __ffma2_rn(p, f, make_float2(1.0000001f, 1.0000001f));
  return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

template <typename T, typename KvT, int D>
__global__ void __launch_bounds__(kMThreads, 2)
    key_mass_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const MassParams p, int split, int* err) {
  using S = MassSmem<D>;
  constexpr int kHalves = D / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) record_error(err, kDevErrSmemAlign);
    pdl_wait();
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sQ = smem + S::kKBytes;
  float* s_nls = reinterpret_cast<float*>(sQ + S::kStages * S::kQBytes);  // [2][kMR] -lse
  int* s_pos = reinterpret_cast<int*>(s_nls + 2 * kMR);                   // [2][kMR]
  float* s_sum = reinterpret_cast<float*>(s_pos + 2 * kMR);               // [2][kMK]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_sum + 2 * kMK);
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;
  uint64_t* s_empty = s_full + 2;
  uint64_t* mma_done = s_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // key tile-major, first keys first: with causal rows these have the most work
  const int bh = blockIdx.x / split, part = blockIdx.x % split, b = bh / (int)p.Hkv, h = bh - b * (int)p.Hkv;
  const int64_t cap = p.mp * p.ps;
  const int k0 = (int)blockIdx.y * kMK;
  // this thread's page, asked for beside the context length, not after it
  int pid = -1;
  uint32_t key_off = 0;
  if (warp < 8 && k0 + (int)(threadIdx.x & 127) < cap) {
    const uint32_t my_key = (uint32_t)k0 + (threadIdx.x & 127), page = my_key / (uint32_t)p.ps;
    key_off = my_key - page * (uint32_t)p.ps;
    pid = __ldg(&p.block_table[(int64_t)b * p.mp + page]);
  }
  const int ctx = p.context_lens[b];
  int64_t end64 = ctx < cap ? ctx : cap;
  if (p.len < end64) end64 = p.len;
  const int end = (int)end64;
  if (k0 >= end) {  // the whole cluster
    // The next kernel waits for this one alone, so this one ends after the attention kernel also
    // when no sequence has a key: the first tile's CTAs wait in any case, here or below.
    if (k0 == 0) pdl_wait();
    return;
  }
  // rows (per run) that see some key of the tile
  const int L = (int)p.L, base_pos = ctx - L;
  const bool by_head = L >= 64;  // else the g * L rows of the kv head are one run
  int lo = 0, hi = by_head ? L : (int)(p.g * p.L);
  if (by_head) {
    if (p.causal && k0 - base_pos > lo) lo = k0 - base_pos;
    if (p.window > 0 && k0 >= p.sinks) {  // pos <= key + window - 1 for the tile's last key
      const int64_t last = (int64_t)k0 + kMK - 1 + p.window - 1 - base_pos;
      if (last + 1 < hi) hi = last + 1 > 0 ? (int)(last + 1) : 0;
    }
  }
  const int n_rows = hi > lo ? hi - lo : 0;
  const int per_run = (n_rows + kMR - 1) / kMR;
  const int runs = by_head ? (int)p.g / split : 1;  // this CTA's heads: part * runs ..
  const int n_tiles = per_run * runs;
  // Walk of the tiles in order: run by run, `in` rows into the run.
  struct Walk {
    int base, in;  // the run's first row of the kv head; rows of the run before this tile
  };
  const Walk first{part * runs * (by_head ? L : 0) + lo, 0};
  auto step = [&](Walk& w) {
    w.in += kMR;
    if (w.in >= n_rows) {
      w.in = 0;
      w.base += L;
    }
  };

  auto load_q = [&](int s, const Walk& w) {
    mbar_arrive_expect_tx(&q_full[s], S::kQBytes);
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf)
      tma_load_3d(sQ + s * S::kQBytes + hf * (kMR * 128), &tm_q, hf * 64, w.base + w.in, bh, &q_full[s]);
  };
  if (threadIdx.x == 8 * 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    Walk w = first;
    for (int t = 0; t < 2 && t < n_tiles; ++t, step(w)) load_q(t, w);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kMCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // K: lane = key for the page lookup, then warps w and w + 4 copy their 32 rows with kLanes
  // lanes a row into the swizzled K-major layout the MMA reads (row r's 16-byte chunk c of a
  // 64-element half at r * 128 + ((c ^ (r & 7)) << 4)); int8 becomes T exactly and its scale
  // multiplies the scores.  Unmapped and out-of-range keys are zero.
  float kf = p.scale_log2;
  bool mapped = false;
  if (warp < 8) {
    const int key = k0 + (int)(threadIdx.x & 127);
    int64_t row = -1;
    if (key < end && pid >= 0 && pid < p.P) row = ((int64_t)pid * p.Hkv + h) * p.ps + key_off;
    mapped = row >= 0;
    if (std::is_same<KvT, int8_t>::value && mapped) kf *= load_dyn(p.ks, row, p.scale_dtype);
    constexpr int kLanes = D * (int)sizeof(KvT) / 16;  // lanes a row, and steps
    constexpr int kRows = 32 / kLanes;                 // rows a step
    const int sub = lane / kLanes, c = lane % kLanes;
    constexpr int kHalf = kLanes / 2;                  // steps of each of the two warps
    const int i0 = (warp >> 2) * kHalf;
    uint4 v[kHalf];
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int64_t src = __shfl_sync(0xffffffffu, row, (i0 + i) * kRows + sub);
      v[i] = src >= 0 ? __ldcs(reinterpret_cast<const uint4*>(static_cast<const KvT*>(p.k) + src * D) + c)
                      : make_uint4(0u, 0u, 0u, 0u);
    }
    auto put = [&](int r, int ch, uint4 x) {
      *reinterpret_cast<uint4*>(sK + (ch >> 3) * (kMK * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x;
    };
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int r = (warp & 3) * 32 + (i0 + i) * kRows + sub;
      if constexpr (std::is_same<KvT, int8_t>::value) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t pair = w[x >> 1] >> (16 * (x & 1));
          o[x] = cvt_pack<T>((float)(int8_t)(pair & 0xFF), (float)(int8_t)((pair >> 8) & 0xFF));
        }
        put(r, 2 * c, make_uint4(o[0], o[1], o[2], o[3]));
        put(r, 2 * c + 1, make_uint4(o[4], o[5], o[6], o[7]));
      } else {
        put(r, c, v[i]);
      }
    }
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 8) {
    // -------------------------------------------------------------- Q copies
    if (lane == 0) {
      bool ok = true;
      int issued = n_tiles < 2 ? n_tiles : 2;
      Walk w = first;
      step(w);
      step(w);
      for (int t = 2; t < n_tiles; ++t) {
        if (!mbar_wait(&q_empty[t & 1], (uint32_t)(((t >> 1) & 1) ^ 1)) || *(volatile int*)abort_flag != 0) {
          ok = false;
          break;
        }
        load_q(t & 1, w);
        step(w);
        issued = t + 1;
      }
      if (!ok) {
        record_error(err, kDevErrEmptyWait);
        *(volatile int*)abort_flag = 1;
      }
      for (int s = 0; s < 2 && s < issued; ++s) {  // every copy lands before the CTA exits
        const int last = s + ((issued - 1 - s) / 2) * 2;
        if (!mbar_wait(&q_full[s], (uint32_t)((last >> 1) & 1))) record_error(err, kDevErrDrainWait);
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // -------------------------------------------------------------- MMAs
    const uint32_t id = idesc<T>(false, kMR);
    const uint64_t dk = smem_desc(smem_u32(sK), 16, 1024), dq = smem_desc(smem_u32(sQ), 16, 1024);
    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t & 1;
      if (!warp_wait(&q_full[s], (uint32_t)((t >> 1) & 1)) ||
          (t >= 2 && !warp_wait(&s_empty[s], (uint32_t)(((t >> 1) & 1) ^ 1)))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t dqs = dq + (uint64_t)((s * S::kQBytes) >> 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t off = (uint64_t)(((ks >> 2) * (kMR * 128) + (ks & 3) * 32) >> 4);
        mma_f16_warp(tmem + (uint32_t)(s * kMR), dk + off, dqs + off, id, ks > 0 ? 1u : 0u);
      }
      mma_commit_warp(&s_full[s]);
      mma_commit_warp(&q_empty[s]);
    }
    if (!ok && lane == 0) {
      record_error(err, kDevErrMmaWait);
      *(volatile int*)abort_flag = 1;
    }
    __syncwarp();
    mma_commit_warp(mma_done);
  } else {
    // -------------------------------------------------------------- exponentials
    // Warps 0-3 take the even tiles, warps 4-7 the odd ones: with two CTAs per SM four warps
    // a scheduler, which hide the tensor-memory loads and the exponentials' latency.
    const int wg = warp >> 2, r = threadIdx.x & 127, key = k0 + r;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int k_last = (k0 + kMK < end ? k0 + kMK : end) - 1;
    const int64_t row_base = (int64_t)bh * p.g * p.L;  // of lse: the kv head's rows are contiguous
    auto row_lse = [&](const Walk& w) -> float {
      return w.in + r < n_rows ? -__ldcg(&p.lse[row_base + w.base + w.in + r]) : -INFINITY;
    };
    pdl_wait();  // K is in shared memory and the first products are on their way: now the log-sum-exps
    Walk w = first;
    if (wg) step(w);
    float next = wg < n_tiles ? row_lse(w) : 0.f;
    float2 acc[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] = make_float2(0.f, 0.f);
    const float2 kf2 = make_float2(kf, kf);
    const bool sink = key < p.sinks;
    bool ok = true;
    const int s = wg;  // the accumulator of this group's tiles
    const uint32_t tS = tmem + lane_base + (uint32_t)(s * kMR);
    float* nls = s_nls + s * kMR;
    int* ps = s_pos + s * kMR;
    for (int t = wg; t < n_tiles; t += 2) {
      const Walk now = w;
      const int rows = n_rows - now.in < kMR ? n_rows - now.in : kMR;
      step(w);
      step(w);
      named_barrier(1 + wg, 128);  // every thread of the group is done with the buffer's last tile
      nls[r] = next;
      if (!by_head) ps[r] = base_pos + (now.in + r) % L;
      if (t + 2 < n_tiles) next = row_lse(w);
      named_barrier(1 + wg, 128);
      // does every row of the tile see every key of the CTA?
      const int pos_lo = by_head ? base_pos + lo + now.in : base_pos;
      const int pos_hi = by_head ? pos_lo + rows - 1 : ctx - 1;
      const bool all = (!p.causal || k_last <= pos_lo) &&
                       (p.window == 0 || k_last < p.sinks || (int64_t)k0 > (int64_t)pos_hi - p.window);
      if (!warp_wait(&s_full[s], (uint32_t)((t >> 1) & 1))) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (all && rows == kMR) {
#pragma unroll 1
        for (int c = 0; c < kMR; c += 32) {
          float v[32];
          tmem_ld32(tS + (uint32_t)c, v);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float4 l4 = *reinterpret_cast<const float4*>(nls + c + 4 * x);
            const float2 z0 = __ffma2_rn(make_float2(v[4 * x], v[4 * x + 1]), kf2, make_float2(l4.x, l4.y));
            const float2 z1 = __ffma2_rn(make_float2(v[4 * x + 2], v[4 * x + 3]), kf2, make_float2(l4.z, l4.w));
            const float2 e0 = (kPolyMask >> x) & 1 ? exp2_poly(z0) : make_float2(ex2_ftz(z0.x), ex2_ftz(z0.y));
            acc[(2 * x) & 3] = __fadd2_rn(acc[(2 * x) & 3], e0);
            acc[(2 * x + 1) & 3] = __fadd2_rn(acc[(2 * x + 1) & 3], make_float2(ex2_ftz(z1.x), ex2_ftz(z1.y)));
          }
        }
      } else {
        // Columns [c_lo, c_hi) of a run see this key (those from `rows` on hold another head's rows);
        // rows of several heads look their position up.
        const int64_t w64 = p.window > 0 && !sink ? p.window : INT64_MAX / 4;
        const int64_t c_hi64 = (int64_t)key + w64 - pos_lo;
        const int c_lo = p.causal ? key - pos_lo : INT32_MIN, c_hi = c_hi64 < rows ? (int)c_hi64 : rows;
#pragma unroll 1
        for (int c0 = 0; c0 < rows; c0 += 32) {
          float sv[32];
          tmem_ld32(tS + (uint32_t)c0, sv);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            bool seen;
            if (by_head) {
              seen = c0 + x >= c_lo && c0 + x < c_hi;
            } else {
              const int pos = ps[c0 + x];
              seen = (!p.causal || key <= pos) && (int64_t)key > (int64_t)pos - w64;
            }
            const float e = seen ? ex2_ftz(fmaf(sv[x], kf, nls[c0 + x])) : 0.f;
            if (x & 1) acc[(x >> 1) & 3].y += e; else acc[(x >> 1) & 3].x += e;
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&s_empty[s]);
    }
    if (!ok && lane == 0) {
      record_error(err, kDevErrFullWait);
      *(volatile int*)abort_flag = 1;
    }
    const float2 a01 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
    s_sum[wg * kMK + r] = mapped ? a01.x + a01.y : 0.f;
  }
  // the two groups' and the cluster's sums, always added in the same order
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (split > 1) cluster.sync(); else __syncthreads();
  const int key = k0 + (int)threadIdx.x;
  if (part == 0 && threadIdx.x < kMK && key < end) {
    float sum = s_sum[threadIdx.x] + s_sum[kMK + threadIdx.x];
    for (int x = 1; x < split; ++x) {
      const float* other = cluster.map_shared_rank(s_sum, x);
      sum += other[threadIdx.x] + other[kMK + threadIdx.x];
    }
    float* m = p.mass + b * p.stride_b + h * p.stride_h + key;
    *m = (key < base_pos ? *m : 0.f) + sum;
  }
  if (split > 1) cluster.sync();  // the sums stay until they have been read

  if (warp == 9 && lane == 0) {
    if (!mbar_wait(mma_done, 0)) record_error(err, kDevErrMmaWait);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMCols) : "memory");
}

template <typename T, typename KvT, int D>
int launch_mass_sm100(const PagedArgs& a, const MassParams& p, int64_t keys, cudaStream_t s) {
  using S = MassSmem<D>;
  auto kern = key_mass_sm100_kernel<T, KvT, D>;
  static std::mutex mu;
  static uint64_t done = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !(done & (1ull << dev))) {
      const int st = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes),
                                "paged_attention: key mass cudaFuncSetAttribute");
      if (st != NVM_OK) return st;
      if (dev < 64) done |= 1ull << dev;
    }
  }
  const CUtensorMapDataType dt =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t rows = (uint64_t)(p.g * p.L);
  const uint64_t qd[3] = {(uint64_t)D, rows, (uint64_t)(p.B * p.Hkv)};
  const uint64_t qs[2] = {D * 2, rows * D * 2};
  const uint32_t qb[3] = {64u, (uint32_t)kMR, 1u};
  CUtensorMap tq;
  const int st = encode_tmap(&tq, dt, 3, a.q, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != NVM_OK) return st;
  // CTAs per cluster: the smallest divisor of the group's heads that makes three CTAs an SM,
  // enough to even out the causal rows (2 x 2048 tokens, 32/8 heads: 512 CTAs 174 us with the
  // attention, 256 CTAs 188 us, 1024 CTAs 182 us, where the start of a CTA weighs more).
  int split = 1;
  const int64_t key_tiles = (keys + kMK - 1) / kMK;
  if (p.L >= 64)
    for (int x = 2; x <= 8 && key_tiles * a.B * a.Hkv * split < 3 * 148; ++x)
      if (p.g % x == 0) split = x;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * split), (unsigned)key_tiles);
  cfg.blockDim = dim3(kMThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = s;
  // Programmatic launch: its CTAs take slots as the attention kernel's last wave ends, and have K
  // in shared memory when that kernel is done (a scored prompt of 2 x 2048: 162 -> 152 us; the
  // kernels that only wait, the scores' and the compaction's, gained nothing by it).
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, tq, p, split, device_error_word()),
                    "paged_attention: key mass kernel launch");
}

template <typename T>
int launch_mass_typed(const PagedArgs& a, const MassParams& p, int64_t keys, cudaStream_t s) {
  if (a.kv_dtype == NVM_I8)
    return a.D == 64 ? launch_mass_sm100<T, int8_t, 64>(a, p, keys, s) : launch_mass_sm100<T, int8_t, 128>(a, p, keys, s);
  return a.D == 64 ? launch_mass_sm100<T, T, 64>(a, p, keys, s) : launch_mass_sm100<T, T, 128>(a, p, keys, s);
}

bool force_generic() {
  const char* v = env_get("NVM_ATTN_FORCE_GENERIC");
  return v != nullptr && v[0] != '\0' && v[0] != '0';
}

// 16-bit queries over pages of their type or int8; the kernel counts keys, rows and
// positions in 32 bits.
bool mass_sm100_eligible(const PagedArgs& a) {
  if (a.q_dtype != NVM_F16 && a.q_dtype != NVM_BF16) return false;
  if (a.kv_dtype != a.q_dtype && a.kv_dtype != NVM_I8) return false;
  if (a.D != 64 && a.D != 128) return false;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a.q) || !al16(a.k_pages)) return false;
  const int64_t lim = INT32_MAX / 2;
  return a.B * a.Hq < lim && a.Hq / a.Hkv * a.L < lim && a.page_size < lim && a.max_pages < lim &&
         a.max_pages * a.page_size < int64_t(65535) * kMK;
}

}  // namespace

int launch_key_mass(const PagedArgs& a, const KeyMassArgs& m, const MmaPlan* plan, const void* ws, bool tensor_cores,
                    cudaStream_t s) {
  MassParams p{};
  p.q = a.q; p.k = a.k_pages; p.ks = a.k_scales; p.block_table = a.block_table; p.context_lens = a.context_lens;
  p.lse = a.lse; p.mass = m.mass; p.stride_b = m.stride_b; p.stride_h = m.stride_h; p.len = m.len;
  p.q_dtype = a.q_dtype; p.kv_dtype = a.kv_dtype; p.scale_dtype = a.scale_dtype;
  p.B = a.B; p.Hq = a.Hq; p.Hkv = a.Hkv; p.L = a.L; p.D = a.D; p.P = a.P; p.ps = a.page_size; p.mp = a.max_pages;
  p.g = a.Hq / a.Hkv;
  p.scale_log2 = a.scale * kLog2e;
  p.causal = a.is_causal; p.window = a.window; p.sinks = a.sinks;
  int64_t keys = a.max_pages * a.page_size;
  if (m.len < keys) keys = m.len;
  if (keys <= 0 || a.B * a.Hkv == 0) return NVM_OK;
  if (a.scores != nullptr) {
    const uint8_t* w = static_cast<const uint8_t*>(ws);
    ScoreParams sp{a.scores, a.defer ? reinterpret_cast<const float2*>(w + mma_ws_ml()) : nullptr,
                   reinterpret_cast<const float*>(w + mma_ws_o(*plan)), a.out, a.out_dtype,
                   plan->chunk_tiles * plan->n_chunks * 16, plan->n_chunks, plan->chunk_tiles, (int)(p.g * p.L)};
    const int64_t per = 256 * kScoreKeys;
    p.blocks = (sp.v_keys + per - 1) / per + (a.defer ? 1 : 0);  // one more: the merge
    if (p.blocks * a.B * a.Hkv > INT32_MAX) return fail(NVM_ERR_UNSUPPORTED, "paged_attention: too many keys for key_mass");
    const dim3 grid((unsigned)(p.blocks * a.B * a.Hkv));
    auto kern = a.defer ? key_mass_scores_kernel<8, true> : key_mass_scores_kernel<8, false>;
    if (sp.rows <= 2) kern = a.defer ? key_mass_scores_kernel<2, true> : key_mass_scores_kernel<2, false>;
    else if (sp.rows <= 4) kern = a.defer ? key_mass_scores_kernel<4, true> : key_mass_scores_kernel<4, false>;
    else if (sp.rows <= 6) kern = a.defer ? key_mass_scores_kernel<6, true> : key_mass_scores_kernel<6, false>;
    kern<<<grid, 256, 0, s>>>(p, sp);
    return check_cuda(cudaGetLastError(), "paged_attention: key mass kernel launch");
  }
  if (!force_generic() && mass_sm100_eligible(a))
    return a.q_dtype == NVM_F16 ? launch_mass_typed<__half>(a, p, keys, s) : launch_mass_typed<__nv_bfloat16>(a, p, keys, s);
  int64_t bx = (keys + kGenWarps - 1) / kGenWarps;
  if (bx > 65536) bx = 65536;
  if (bx * a.B * a.Hkv > INT32_MAX) bx = INT32_MAX / (a.B * a.Hkv);
  if (bx < 1) return fail(NVM_ERR_UNSUPPORTED, "paged_attention: too many sequences for key_mass");
  p.blocks = bx;
  // the tensor-core attention kernels take q in the pages' type (f16 over int8 pages)
  p.q_round = !tensor_cores ? NVM_F32 : a.kv_dtype == NVM_I8 ? NVM_F16 : a.kv_dtype;
  const dim3 grid((unsigned)(bx * a.B * a.Hkv));
  key_mass_generic_kernel<<<grid, kGenWarps * 32, 0, s>>>(p);
  return check_cuda(cudaGetLastError(), "paged_attention: key mass kernel launch");
}

}  // namespace nvm
