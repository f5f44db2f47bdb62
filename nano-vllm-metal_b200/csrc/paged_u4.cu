// paged_u4.cu -- paged attention over a cache held in 4 bits (u4.cuh has the row format).
//
// Semantics are those of the other paged kernels: positions at or past min(ctx, max_pages * page_size),
// holes (page id < 0 or >= P) and, with the causal limit, keys after l + ctx - L are skipped; a row that
// sees nothing is zero, and a key that no row sees has no influence whatever it holds.
//
// Mathematics.  With K = s c + z and V = s' c' + z' (one pair a group of 64 elements) a score is
//   q.k = sum over groups of s (q . c) + z (sum of q),
// and an output element of group g is (sum p s'_g c' + sum p z'_g) / sum p: codes enter the matrix
// instructions as they are, scales and offsets act on scores and weights.  A code needs no conversion:
// bits 0-3 of a 16-bit word are the f16 subnormal code * 2^-24 and bits 4-7 code * 2^-20, so one logic
// operation makes two operands (and one shift serves the upper bytes), exactly and without a bias that
// sums would have to lose again; the powers of two go into the queries and into the output.
// Queries are held in f16, each row scaled by a power of two (exact for 16-bit queries).
//
// Weights are 2^(t - M), t the base-2 score and M a reference of the row's near the largest t so far; their sum and
// that of p z' are fp32.  Multiplied by s' they are held in f16, in a unit of the row's and the group's own: F, a
// power of two, brings the largest product so far to about 1, and f16 holds what matters to 11 bits however the
// values of the keys that are attended to, or the two groups of a key, differ in size.  M and F move only where a
// weight or a product passes them by kSlack, which one vote over a tile's largest weights and scales finds, and
// only by keys that the row sees.  (One reference for weights and both groups took 3 to 5 % less time, and lost
// the smaller group's bits from a ratio of 2^14, all of them at 2^26.)
//
// The floor of a decode step is HBM: 144 bytes a key and kv head (D = 128).  64 requests of 2K-16K keys, 32/8
// heads, take 129 us, 0.78 of a copy's rate (48 of 4K-12K, 64/8 heads, f16: 96 us, 0.71), in a graph of a dozen
// calls; in runs of hundreds, where the power limit lowers the clocks, 139 to 142 (101).  The variants below are
// compared in such runs.  What bounds it is the latency of the instructions: about 500 a tile of 32 keys and warp
// (unpacking 160, weights, their references and sums 230, matrix instructions 36, copies 60), 12 warps an SM at 168
// registers, issue slots 51 % busy.  Tiles come by 16-byte asynchronous copies, a ring to each warp, so that no
// warp waits for another inside a unit.
#include <algorithm>
#include <type_traits>

#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kWarps = 4;    // 2: a long context 43 us for 33; 8: 64 requests 148 us for 139, 5 tokens 113 for 103
constexpr int kTile = 32;    // keys of a stage, one page lookup a lane
constexpr int kStages = 2;   // of each warp's own ring: one tile is copied while one is worked on
// Blocks an SM holds.  One tile of rows: of 64 elements four at 124 registers (three: 30.7 us for 28.7); of 128
// three, whose 168 registers hold what four spill (64 requests 139 us, four 146, two 162).  Two tiles: two
// (5 tokens 103 us, three 108).
constexpr int blocks_of(int64_t D, int tiles) { return tiles == 2 ? 2 : D == 128 ? 3 : 4; }
constexpr int kStep = kWarps * kTile;  // keys that a block takes at a time, the unit that work is dealt in
constexpr int kUnitCost = 3;  // steps that beginning and ending a unit takes the time of (0: 64 requests 146 us for 139, 5 tokens 125 for 103; 6: 142, 100)
constexpr int kFan = 16;     // partial results that are joined at a time (8: one request 14.4 us for 13.0; 40: one of 90K-130K keys 35.0 for 33.0)
constexpr float kSlack = 1024.0f;   // how far a weight may pass 2^M, and a weight times a scale its unit
constexpr float kLeast = 0x1p-100f;  // least scale that a key's values count as
constexpr float kNoKeys = -0x1p127f;  // M of a row that has seen no key
// From scores of this size on the exact product of score and factor is further from M, the rounded one, than a
// weight may pass it by (4 here, 128 at 2^31, which is infinity): such a row's factor becomes a power of two, whose
// product is exact.  Scores of this size are 8 apart, and ordered as before.
constexpr float kFar = 0x1p27f;

template <int D>
struct Ring {
  static constexpr int kGroups = D / kU4Group;
  static constexpr int kRow = D / 2;  // bytes of a row's codes
  static constexpr int kV = kTile * kRow, kKs = 2 * kV, kVs = kKs + kTile * 4 * kGroups;
  static constexpr int kStage = kVs + kTile * 4 * kGroups;
  static constexpr int kWarp = kStages * kStage;
};

struct U4Params {
  const void* q;
  const uint8_t* kp;
  const uint8_t* vp;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* block_table;
  const int32_t* context_lens;
  void* out;
  float2* part_ml;  // [2 * blocks][rows of a unit]: (M, sum of weights)
  float* part_o;    // [2 * blocks][rows of a unit][D]
  int* tickets;     // [3 * blocks], zero between calls: of groups by their leader's place, of units by their first block
  int q_dtype, out_dtype, causal;
  int q_fast;  // rows of 16-bit numbers on 16-byte boundaries
  int B, Hkv, L, rows, row_block0, row_blocks, P, ps, mp;  // the launch's row blocks of a (request, kv head)
  U4Some some;
  FastDiv by_ps;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(there ? kBytes : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 operations as one: d = a * b + c, d = a * b, d = a + b
__device__ __forceinline__ void fma2(float a0, float a1, float b0, float b1, float c0, float c1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float a0, float a1, float b0, float b1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float a0, float a1, float b0, float b1, float& d0, float& d1) {
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// the codes in bits 0-3 and 4-7 of both halves, as f16 subnormals
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00f000f0u; }
constexpr float kLowUnit = 0x1p24f, kHighUnit = 0x1p20f;  // what undoes their size

// The 16-byte parts of rows are swapped so that the eight rows of a matrix load touch every bank once.
template <int D>
__device__ __forceinline__ int swizzle(int key) {
  return D == 128 ? key >> 1 & 3 : key >> 2 & 1;
}

// (scale, offset) of a key's groups.
template <typename T, int kGroups>
struct Pairs {
  float s[kGroups], z[kGroups];
  __device__ __forceinline__ void load(uint32_t addr) {
    uint32_t w[2];
    if constexpr (kGroups == 2) {
      const uint2 v = lds64(addr);
      w[0] = v.x;
      w[1] = v.y;
    } else {
      w[0] = lds32(addr);
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float2 p = u4_pair<T>(w[g]);
      s[g] = p.x;
      z[g] = p.y;
    }
  }
};

// Keys of a request that some query row may see, in steps of kStep; one at least, so that every row
// is written (kSome: none where no row is to be).
template <bool kSome>
__device__ __forceinline__ int steps_of(const U4Params& p, int b) {
  if (kSome && __ldg(p.some.some + b) == 0) return 0;
  const int keys = min(__ldg(p.context_lens + b), p.mp * p.ps);
  return max(1, (keys + kStep - 1) / kStep);
}

// Joins `count` partial results (M, sum, output in units of 2^M) of a unit, the k-th in place of(k), into
// the output's rows in `chosen` or, with `to` >= 0, into that place.  All threads of the block; `scratch` holds
// count x kRows.
template <int D, int kRows, typename Of>
__device__ __forceinline__ void join(const U4Params& p, float2* scratch, int count, Of&& of, int rows, size_t out_row0, int to,
                                     uint32_t chosen) {
  for (int i = threadIdx.x; i < count * kRows; i += kWarps * 32)
    scratch[i] = __ldcg(p.part_ml + (size_t)of(i / kRows) * kRows + i % kRows);
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += kWarps * 32) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float top = kNoKeys, sum = 0.0f;
    for (int k = 0; k < count; ++k) top = fmaxf(top, scratch[k * kRows + row].x);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int k = 0; k < count; ++k) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((size_t)of(k) * kRows + row) * D + d));
      const float2 ml = scratch[k * kRows + row];
      const float f = ex2(ml.x - top);
      sum = fmaf(f, ml.y, sum);
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    }
    if (to >= 0) {
      *reinterpret_cast<float4*>(p.part_o + ((size_t)to * kRows + row) * D + d) = o;
      if (d == 0) p.part_ml[(size_t)to * kRows + row] = make_float2(top, sum);
    } else if (chosen >> row & 1) {
      const int64_t at = (int64_t)(out_row0 + row) * D + d;
      const float inv = sum == 0.0f ? 0.0f : __frcp_rn(sum);
      store_dyn(p.out, at, p.out_dtype, o.x * inv);
      store_dyn(p.out, at + 1, p.out_dtype, o.y * inv);
      store_dyn(p.out, at + 2, p.out_dtype, o.z * inv);
      store_dyn(p.out, at + 3, p.out_dtype, o.w * inv);
    }
  }
}

// A unit is kTiles x 8 query rows of one (request, kv head).  The units' keys, in steps of kStep, form
// one line that is dealt to the blocks in equal parts, so that requests of any lengths load every SM
// alike; a block takes the units on its part one after another.  Its warps walk tiles of 32 keys, each
// through a ring of its own, and are joined in shared memory.  A unit that several blocks share is
// joined by the last of them (in groups of kFan, then the groups).  kSome: only the rows that U4Some names
// are computed and written.
template <typename T, int D, int kTiles, bool kSome>
__global__ void __launch_bounds__(kWarps * 32, blocks_of(D, kTiles)) paged_u4_kernel(const U4Params p) {
  using R = Ring<D>;
  constexpr int G = R::kGroups, kRows = 8 * kTiles;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][kRows];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;

  // The line's length, this block's part of it and the request that the part begins in.  Every unit
  // counts kUnitCost steps more than it has (where there is more than a step a block): that long a block
  // is busy with beginning and ending one.  Lane i adds up the requests [i * per, (i + 1) * per).
  const int heads = p.Hkv * p.row_blocks;  // units of a request
  const int per = (p.B + 31) / 32;
  int upto = 0, requests = max(min(per, p.B - lane * per), 0);
  for (int i = lane * per; i < min((lane + 1) * per, p.B); ++i) {
    const int n = steps_of<kSome>(p, i);
    upto += n;
    if (kSome && n == 0) --requests;
  }
  const int real = __reduce_add_sync(0xffffffffu, upto) * heads;
  const int cost = real > (int)gridDim.x ? kUnitCost : 0;
  upto += cost * requests;
  const int mine = upto;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const int total = __shfl_sync(0xffffffffu, upto, 31) * heads, blocks = min((int)gridDim.x, total);
  if ((int)blockIdx.x >= blocks) return;
  // the first `more` blocks take share + 1 steps, the others share; step x is in block_of(x)
  const int share = total / blocks, more = total - share * blocks;
  auto block_of = [&](int x) -> int {
    return x < more * (share + 1) ? x / (share + 1) : more + (x - more * (share + 1)) / share;
  };
  int pos = (int)blockIdx.x * share + min((int)blockIdx.x, more);
  const int pos_end = pos + share + ((int)blockIdx.x < more);
  const int in_lane = __ffs(__ballot_sync(0xffffffffu, upto * heads > pos)) - 1;
  int b = in_lane * per, request_at = __shfl_sync(0xffffffffu, upto - mine, in_lane) * heads;  // where request b begins
  int steps = steps_of<kSome>(p, b);

  while (pos < pos_end) {
  while ((kSome && steps == 0) || pos >= request_at + (steps + cost) * heads) {
    if (!kSome || steps > 0) request_at += (steps + cost) * heads;
    steps = steps_of<kSome>(p, ++b);
  }
  const int in_request = (pos - request_at) / (steps + cost);
  const int unit_at = request_at + in_request * (steps + cost) + cost;  // its first step
  if (unit_at >= pos_end) break;
  const int step0 = max(pos - unit_at, 0), step1 = min(steps, pos_end - unit_at);
  pos = unit_at + step1;
  const int kvh = in_request / p.row_blocks, rb = p.row_block0 + in_request - kvh * p.row_blocks, bh = b * p.Hkv + kvh;
  const int row0 = rb * kRows, rows = min(kRows, p.rows - row0);
  const int ctx = __ldg(p.context_lens + b), limit = min(ctx, p.mp * p.ps);
  // keys that the unit's rows see: [0, most) by some row, [0, least) by every row
  int most = limit, least = limit;
  if (p.causal && p.L > 1) {
    int lo = row0 % p.L, hi = (row0 + rows - 1) % p.L;
    if (rows >= p.L || lo > hi) {
      lo = 0;
      hi = p.L - 1;
    }
    most = min(limit, hi + ctx - p.L + 1);
    least = min(limit, lo + ctx - p.L + 1);
  }
  most = max(most, 0);
  const int begin = min(step0 * kStep, most), end = min(step1 * kStep, most);

  const size_t out_row0 = (size_t)bh * p.rows + row0;
  uint32_t chosen = 0xffffffffu;
  if constexpr (kSome) {
    const uint32_t first = __ldg(p.some.first + bh);
    bool mine = false;
    if (lane < rows) {
      const int see = p.causal ? min(limit, (row0 + lane) % p.L + ctx - p.L + 1) : limit;
      mine = (first != 0 && INT32_MAX - (int)first < see) || __ldg(p.some.rows + out_row0 + lane) != 0;
    }
    chosen = __ballot_sync(0xffffffffu, mine);
    if (chosen == 0) continue;
  }
  uint8_t* ring = smem + warp * R::kWarp;
  const uint32_t ring_at = smem_u32(ring);
  const int32_t* bt = p.block_table + (size_t)b * p.mp;

  auto page_of_key = [&](int key) -> int {
    if (key >= end) return -1;
    const int pid = __ldg(bt + p.by_ps((uint32_t)key));
    return pid < p.P ? pid : -1;
  };
  // Copies the tile whose first key is k0 (a lane's key lies in page pid) into a stage and says which of
  // its keys are there.  The others read codes of the pool's first row, which are numbers in any case,
  // with scales and offsets of zero.
  constexpr int kParts = R::kRow / 16, kKeysAStep = 32 / kParts;
  const uint8_t* k_lane = p.kp + lane % kParts * 16;
  const uint8_t* v_lane = p.vp + lane % kParts * 16;
  const uint32_t dst_lane = ring_at + lane / kParts * R::kRow +
                            ((lane % kParts ^ swizzle<D>(lane / kParts)) << 4);
  auto issue = [&](int k0, int pid, int stage) -> uint32_t {
    const uint32_t page = p.by_ps((uint32_t)(k0 + lane));
    const uint32_t off = (uint32_t)(k0 + lane) - page * (uint32_t)p.ps;
    const uint32_t row = pid < 0 ? 0u : ((uint32_t)pid * p.Hkv + kvh) * p.ps + off;
    const uint32_t dst = dst_lane + stage * R::kStage;
#pragma unroll
    for (int i = 0; i < kTile / kKeysAStep; ++i) {
      const uint32_t krow = __shfl_sync(0xffffffffu, row, i * kKeysAStep + lane / kParts);
      cp_async16(dst + i * kKeysAStep * R::kRow, k_lane + (uint64_t)krow * R::kRow);
      cp_async16(dst + R::kV + i * kKeysAStep * R::kRow, v_lane + (uint64_t)krow * R::kRow);
    }
    const uint32_t at = ring_at + stage * R::kStage + lane * 4 * G;
    cp_async_small<4 * G>(at + R::kKs, p.ks + (uint64_t)row * (4 * G), pid >= 0);
    cp_async_small<4 * G>(at + R::kVs, p.vs + (uint64_t)row * (4 * G), pid >= 0);
    return __ballot_sync(0xffffffffu, pid >= 0);
  };

  int k_next = begin + warp * kTile;  // first key of the tile to copy next
  int pid = page_of_key(k_next + lane);
  const int pid1 = page_of_key(k_next + kStep + lane);
  // 16-bit rows on 16-byte boundaries: a lane's elements are on their way before the tile's pages are known
  uint4 raw[kTiles][G][2];
  if (p.q_fast) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          raw[j][g][h] = make_uint4(0, 0, 0, 0);
          if (8 * j + r < rows)
            raw[j][g][h] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (out_row0 + 8 * j + r) * D) +
                                 (g * kU4Group + h * 32 + c * 8) / 8);
        }
  }
  uint32_t there_next = k_next < end ? issue(k_next, pid, 0) : 0;  // the keys of the tile on its way
  cp_async_commit();
  k_next += kStep;
  pid = pid1;

  // Queries as B fragments (lane: row r of each tile of 8; of a group, elements 8c to 8c + 7 of each half),
  // scaled per row so that the largest is in [2^10, 2^11), and 16 times that where they meet low codes;
  // kap undoes it and turns scores to base 2.
  uint32_t qf[kTiles][G][4][2];
  float kap[kTiles][2], qsum[kTiles][2][G];  // qsum in units of the scores before kap
  int seen[kTiles][2];  // keys [0, seen) are seen by the lane's rows 2c, 2c + 1
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    float x[G][16], top = 0.0f;
    const int row = 8 * j + r;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (p.q_fast) {
          const uint4 v = raw[j][g][h];
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = p.q_dtype == NVM_BF16 ? u4_pair<__nv_bfloat16>(u[i]) : u4_pair<__half>(u[i]);
            x[g][8 * h + 2 * i] = f.x;
            x[g][8 * h + 2 * i + 1] = f.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            x[g][8 * h + i] = row < rows ? load_dyn(p.q, (int64_t)(out_row0 + row) * D + g * kU4Group + h * 32 + c * 8 + i, p.q_dtype) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[g][8 * h + i]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e2 = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 100);
    float up = __uint_as_float((uint32_t)(127 + 10 - e2) << 23);
    float down = p.scale_log2 * __uint_as_float((uint32_t)(127 - 10 + e2) << 23) * kHighUnit;
    if (down == 0.0f) {  // every score is 0; masks need a factor that is not
      up = 0.0f;
      down = 1.0f;
    }
    float sum[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      sum[g] = 0.0f;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // elements (2h + i, 2h + i + 4) of word w
            const float unit = i == 0 ? up * (kLowUnit / kHighUnit) : up;
            const __half2 v = __floats2half2_rn(x[g][8 * w + 2 * h + i] * unit, x[g][8 * w + 2 * h + i + 4] * unit);
            qf[j][g][2 * w + h][i] = *reinterpret_cast<const uint32_t*>(&v);
            const float2 f = __half22float2(v);
            sum[g] += (f.x + f.y) * (i == 0 ? 1.0f / kLowUnit : 1.0f / kHighUnit);
          }
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kap[j][i] = __shfl_sync(0xffffffffu, down, (2 * c + i) * 4);
#pragma unroll
      for (int g = 0; g < G; ++g) qsum[j][i][g] = __shfl_sync(0xffffffffu, sum[g], (2 * c + i) * 4);
      const int rr = 8 * j + 2 * c + i;
      seen[j][i] = rr >= rows || !p.causal ? limit : min(limit, (p.L == 1 ? 0 : (row0 + rr) % p.L) + ctx - p.L + 1);
    }
  }

  // l and zsum in units of 2^M, acc and wsum of 2^M / F
  float acc[G][4][kTiles][4], wsum[G][kTiles][4], M[kTiles][2], F[kTiles][2][G], l[kTiles][2], zsum[kTiles][2][G];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wsum[g][j][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i][j][e] = 0.0f;
      }
      zsum[j][0][g] = zsum[j][1][g] = 0.0f;
      F[j][0][g] = F[j][1][g] = 1.0f;
    }
    M[j][0] = M[j][1] = kNoKeys;
    l[j][0] = l[j][1] = 0.0f;
  }

  // what a lane addresses in a matrix load of 16 keys: K rows 0-7 in matrices 0 and 1 (the group's halves),
  // 8-15 in 2 and 3; V (transposed) rows 0-7 in matrices 0 and 2, 8-15 in 1 and 3
  uint32_t k_off[G], v_off[G];
  {
    const int m = lane >> 3, k_key = (lane & 7) + 8 * (m >> 1), v_key = (lane & 7) + 8 * (m & 1);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      k_off[g] = k_key * R::kRow + (((2 * g + (m & 1)) ^ swizzle<D>(k_key)) << 4);
      v_off[g] = R::kV + v_key * R::kRow + (((2 * g + (m >> 1)) ^ swizzle<D>(v_key)) << 4);
    }
  }

  int stage = 0;
  for (int k0 = begin + warp * kTile; k0 < end; k0 += kStep) {
    cp_async_wait_all();
    __syncwarp();
    const uint32_t there = there_next;
    if (k_next < end) there_next = issue(k_next, pid, stage ^ 1);
    cp_async_commit();
    k_next += kStep;
    pid = page_of_key(k_next + lane);
    const uint32_t at = ring_at + stage * R::kStage;
    stage ^= 1;

    // x[mt][j][e]: score / kap of key r + 16 mt + 8 (e / 2), row 2c + e % 2 of tile j
    float x[2][kTiles][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      Pairs<T, G> a, d;
      a.load(at + R::kKs + (r + 16 * mt) * 4 * G);
      d.load(at + R::kKs + (r + 16 * mt + 8) * 4 * G);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t k[4];  // words of rows r and r + 8 in the group's halves
        ldsm_x4(at + k_off[g] + 16 * mt * R::kRow, k[0], k[1], k[2], k[3]);
        float dot[kTiles][4];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t u = k[w], v = k[2 + w], u8 = u >> 8, v8 = v >> 8;
          const uint32_t a0[4] = {low_codes(u), low_codes(v), high_codes(u), high_codes(v)};
          const uint32_t a1[4] = {low_codes(u8), low_codes(v8), high_codes(u8), high_codes(v8)};
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            if (w == 0)
              mma_first(dot[j], a0, qf[j][g][0][0], qf[j][g][0][1]);
            else
              mma16816<__half>(dot[j], a0, qf[j][g][2][0], qf[j][g][2][1]);
            mma16816<__half>(dot[j], a1, qf[j][g][2 * w + 1][0], qf[j][g][2 * w + 1][1]);
          }
        }
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float s = e < 2 ? a.s[g] : d.s[g], z = e < 2 ? a.z[g] : d.z[g];
            float o0, o1;
            if (g == 0)
              mul2(z, z, qsum[j][0][g], qsum[j][1][g], o0, o1);
            else
              fma2(z, z, qsum[j][0][g], qsum[j][1][g], x[mt][j][e], x[mt][j][e + 1], o0, o1);
            fma2(s, s, dot[j][e], dot[j][e + 1], o0, o1, x[mt][j][e], x[mt][j][e + 1]);
          }
      }
    }

    const bool masked = there != 0xffffffffu || k0 + kTile > least;
    // key of the tile, and where the keys of a row end
    auto sees = [&](int key, int end_of_row) { return (there >> key & 1) != 0 && k0 + key < end_of_row; };
    if (masked) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = r + 16 * mt + 8 * (e >> 1);
            if (!sees(key, seen[j][e & 1])) x[mt][j][e] = kap[j][e & 1] < 0.0f ? INFINITY : -INFINITY;  // kap * x = -inf
          }
    }

    // weights 2^(t - M); a row whose weight, or whose weight times a scale, passes its unit by kSlack moves to the
    // largest so far (only what the row itself sees moves it, so keys that it does not see leave no trace)
    float w[2][kTiles][4], heavy = 0.0f, size[G];
    {  // the largest scales of the tile's values, of the lane's key first (positive numbers compare as integers)
      Pairs<T, G> v;
      v.load(at + R::kVs + lane * 4 * G);
#pragma unroll
      for (int g = 0; g < G; ++g)
        size[g] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(v.s[g], 0.0f))));
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float u0, u1;
          fma2(kap[j][0], kap[j][1], x[mt][j][e], x[mt][j][e + 1], -M[j][0], -M[j][1], u0, u1);
          w[mt][j][e] = ex2(u0);
          w[mt][j][e + 1] = ex2(u1);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float unit = 1.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) unit = fmaxf(unit, F[j][i][g] * size[g]);
        heavy = fmaxf(heavy, unit * fmaxf(fmaxf(w[0][j][i], w[0][j][2 + i]), fmaxf(w[1][j][i], w[1][j][2 + i])));
      }
    }
    if (__any_sync(0xffffffffu, heavy > kSlack)) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float own = 0.0f, most = -INFINITY, product[G];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              Pairs<T, G> v;
              v.load(at + R::kVs + (r + 16 * mt + 8 * h) * 4 * G);
              float unit = 1.0f;
#pragma unroll
              for (int g = 0; g < G; ++g) unit = fmaxf(unit, F[j][i][g] * v.s[g]);
              own = fmaxf(own, unit * w[mt][j][2 * h + i]);
              most = fmaxf(most, kap[j][i] < 0.0f ? -x[mt][j][2 * h + i] : x[mt][j][2 * h + i]);
            }
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) {
            own = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, o));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          }
          const bool move = own > kSlack;
          float top = fmaxf(M[j][i], fabsf(kap[j][i]) * most);
          if (move && fabsf(top) >= kFar) {  // the row goes on with the power of two below its factor
            const float was = kap[j][i];
            kap[j][i] = __uint_as_float(__float_as_uint(was) & 0xff800000u);
            M[j][i] *= __fdiv_rn(kap[j][i], was);
            top = fmaxf(M[j][i], fabsf(kap[j][i]) * most);
          }
#pragma unroll
          for (int g = 0; g < G; ++g) product[g] = kNoKeys;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              Pairs<T, G> v;
              v.load(at + R::kVs + (r + 16 * mt + 8 * h) * 4 * G);
              const float u = fmaf(kap[j][i], x[mt][j][2 * h + i], -top);
              if (move) w[mt][j][2 * h + i] = ex2(u);
#pragma unroll
              for (int g = 0; g < G; ++g) product[g] = fmaxf(product[g], u + lg2(fmaxf(v.s[g], kLeast)));
            }
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1)
#pragma unroll
            for (int g = 0; g < G; ++g) product[g] = fmaxf(product[g], __shfl_xor_sync(0xffffffffu, product[g], o));
          if (!move) continue;
          const float step = M[j][i] - top, fade = ex2(step);
          M[j][i] = top;
          l[j][i] *= fade;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            // the old unit's logarithm was M - log2 F, in terms of the new M: step - log2 F
            const int was = (int)(__float_as_uint(F[j][i][g]) >> 23) - 127;
            const int now = min(max(__float2int_rd(-fmaxf(step - (float)was, product[g])), -126), 126);
            F[j][i][g] = __uint_as_float((uint32_t)(127 + now) << 23);
            const float fade_g = ex2(step + (float)(now - was));
            zsum[j][i][g] *= fade;
            wsum[g][j][i] *= fade_g;
            wsum[g][j][2 + i] *= fade_g;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              acc[g][t][j][i] *= fade_g;
              acc[g][t][j][2 + i] *= fade_g;
            }
          }
        }
    }

    // The weights' sums, the weights times the values' scales as B fragments, and those times the codes.  What
    // f16 rounds off a weight counts times the code less 8 (the sum of weight * (offset + 8 scale) is exact, and
    // 8 times the sum of the rounded weights, a product with ones, is taken out at the end): half of what it would
    // times the code.  In a masked tile a key that the row does not see counts nothing whatever its values.
    auto values = [&](auto hidden) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t pf[kTiles][G][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = r + 16 * mt + 8 * h;
          Pairs<T, G> v;
          v.load(at + R::kVs + key * 4 * G);
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            const float w0 = w[mt][j][2 * h], w1 = w[mt][j][2 * h + 1];
            add2(l[j][0], l[j][1], w0, w1, l[j][0], l[j][1]);
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const float middle = fmaf(8.0f, v.s[g], v.z[g]);
              float s0, s1;
              mul2(w0, w1, F[j][0][g], F[j][1][g], s0, s1);
              mul2(s0, s1, v.s[g], v.s[g], s0, s1);
              if constexpr (decltype(hidden)::value) {
                if (!sees(key, seen[j][0])) s0 = 0.0f;
                if (!sees(key, seen[j][1])) s1 = 0.0f;
                zsum[j][0][g] += sees(key, seen[j][0]) ? w0 * middle : 0.0f;
                zsum[j][1][g] += sees(key, seen[j][1]) ? w1 * middle : 0.0f;
              } else {
                fma2(w0, w1, middle, middle, zsum[j][0][g], zsum[j][1][g], zsum[j][0][g], zsum[j][1][g]);
              }
              pf[j][g][h] = transpose8x8(pack2<__half>(s0, s1));
            }
          }
        }
        const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t v[4];  // keys (2c, 2c + 1) and (2c, 2c + 1) + 8: elements 4r to 4r + 3 of the group's halves
          ldsm_x4_t(at + v_off[g] + 16 * mt * R::kRow, v[0], v[1], v[2], v[3]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t y = v[2 * half], z = v[2 * half + 1], y8 = y >> 8, z8 = z >> 8;
            const uint32_t a0[4] = {low_codes(y), high_codes(y), low_codes(z), high_codes(z)};
            const uint32_t a1[4] = {low_codes(y8), high_codes(y8), low_codes(z8), high_codes(z8)};
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              mma16816<__half>(acc[g][2 * half][j], a0, pf[j][g][0], pf[j][g][1]);
              mma16816<__half>(acc[g][2 * half + 1][j], a1, pf[j][g][0], pf[j][g][1]);
            }
          }
#pragma unroll
          for (int j = 0; j < kTiles; ++j) mma16816<__half>(wsum[g][j], one, pf[j][g][0], pf[j][g][1]);
        }
      }
    };
    if (masked)
      values(std::true_type{});
    else
      values(std::false_type{});
  }
  cp_async_wait_all();

  // the warp's rows: (M, sum of weights) and sum of weight * value, in units of 2^M
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        l[j][i] += __shfl_xor_sync(0xffffffffu, l[j][i], o);
#pragma unroll
        for (int g = 0; g < G; ++g) zsum[j][i][g] += __shfl_xor_sync(0xffffffffu, zsum[j][i][g], o);
      }
    }
  __syncthreads();  // every warp is done with its ring: the rows go there
  constexpr int kPitch = D + 8;
  float* part = reinterpret_cast<float*>(smem) + warp * kRows * kPitch;
  static_assert(kWarps * kRows * kPitch * 4 <= kWarps * R::kWarp, "the rows fit in the rings");
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 8 * j + 2 * c + i;
      // M in terms of the scores' own factor, also where the warp took a power of two
      const float factor = (__float_as_uint(kap[j][i]) & 0x7fffffu) == 0 ? __uint_as_float((__float_as_uint(p.scale_log2) & 0x7fffffu) | 0x3f800000u) : 1.0f;
      if (r == 0) s_ml[warp][row] = make_float2(M[j][i] * factor, l[j][i]);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float less = -8.0f * wsum[g][j][i], more = zsum[j][i][g];
        const float unit = __uint_as_float((254u << 23) - __float_as_uint(F[j][i][g]));  // 1 / F
        float* dst = part + row * kPitch + g * kU4Group + r * 4;
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<float4*>(dst + 32 * half) = make_float4(
              fmaf(fmaf(kLowUnit, acc[g][2 * half][j][i], less), unit, more),
              fmaf(fmaf(kHighUnit, acc[g][2 * half][j][2 + i], less), unit, more),
              fmaf(fmaf(kLowUnit, acc[g][2 * half + 1][j][i], less), unit, more),
              fmaf(fmaf(kHighUnit, acc[g][2 * half + 1][j][2 + i], less), unit, more));
      }
    }
  __syncthreads();

  // Blocks first .. last share the unit.  A block's partial results: 2 i + 1 of a unit that it begins,
  // 2 i of one that it continues.
  const bool whole = step0 == 0 && step1 == steps;
  const int place = 2 * blockIdx.x + (step0 == 0);
  for (int i = threadIdx.x; i < rows * D; i += kWarps * 32) {
    const int row = i / D, d = i - row * D;
    float top = s_ml[0][row].x, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_ml[w][row].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = s_ml[w][row];
      const float f = ex2(ml.x - top);
      sum = fmaf(f, ml.y, sum);
      o = fmaf(f, reinterpret_cast<const float*>(smem)[(w * kRows + row) * kPitch + d], o);
    }
    if (whole) {
      if (chosen >> row & 1) store_dyn(p.out, (int64_t)(out_row0 + row) * D + d, p.out_dtype, sum == 0.0f ? 0.0f : o * __frcp_rn(sum));
    } else {
      p.part_o[((size_t)place * kRows + row) * D + d] = o;
      if (d == 0) p.part_ml[(size_t)place * kRows + row] = make_float2(top, sum);
    }
  }
  if (!whole) {
    const int first = block_of(unit_at), last = block_of(unit_at + steps - 1);
    const int share = last - first + 1, mine = (int)blockIdx.x - first, group = mine / kFan;
    const int groups = (share + kFan - 1) / kFan, count = min(kFan, share - group * kFan);
    const int leader = first + group * kFan;
    auto place_of = [&](int block) { return 2 * block + (block == first); };
    float2* scratch = reinterpret_cast<float2*>(smem);
    // the last of `n` blocks to come, which finds what the others left
    auto last_of = [&](int* ticket, int n) -> bool {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        s_last = atomicAdd(ticket, 1) == n - 1;
        if (s_last) *ticket = 0;
      }
      __syncthreads();
      const bool yes = s_last != 0;
      if (yes) __threadfence();
      return yes;
    };
    if (last_of(p.tickets + place_of(leader), count)) {
      join<D, kRows>(p, scratch, count, [&](int k) { return place_of(leader + k); }, rows, out_row0,
                     groups > 1 ? place_of(leader) : -1, chosen);
      if (groups > 1 && last_of(p.tickets + 2 * gridDim.x + first, groups))
        join<D, kRows>(p, scratch, groups, [&](int k) { return place_of(first + k * kFan); }, rows, out_row0, -1, chosen);
    }
  }
  __syncthreads();  // the rings are free for the next unit
  }
}

template <typename T, int D, int kTiles, bool kSome = false>
int launch(const U4Params& p, int64_t blocks, cudaStream_t s) {
  constexpr int bytes = kWarps * Ring<D>::kWarp;
  const cudaError_t e = cudaFuncSetAttribute(paged_u4_kernel<T, D, kTiles, kSome>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return check_cuda(e, "paged_attention: cudaFuncSetAttribute");
  paged_u4_kernel<T, D, kTiles, kSome><<<(unsigned)blocks, kWarps * 32, bytes, s>>>(p);
  return check_cuda(cudaGetLastError(), "paged_attention: 4-bit kernel launch");
}

template <typename T>
int launch_d(const U4Params& p, int64_t D, int tiles, int64_t blocks, cudaStream_t s) {
  if (p.some.some != nullptr) return launch<T, 128, 2, true>(p, blocks, s);  // (pages are unpacked for no other shape)
  if (D == 128) return tiles == 1 ? launch<T, 128, 1>(p, blocks, s) : launch<T, 128, 2>(p, blocks, s);
  return tiles == 1 ? launch<T, 64, 1>(p, blocks, s) : launch<T, 64, 2>(p, blocks, s);
}

}  // namespace

U4Plan plan_paged_u4(const PagedArgs& a) {
  U4Plan plan{};
  const int64_t rows = a.Hq / a.Hkv * a.L;
  plan.tiles = rows <= 8 ? 1 : 2;
  plan.row_blocks = (rows + 8 * plan.tiles - 1) / (8 * plan.tiles);
  const int64_t steps = std::max<int64_t>((a.max_pages * a.page_size + kStep - 1) / kStep, 1);
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t most = (int64_t)sms * blocks_of(a.D, plan.tiles), units = a.B * a.Hkv * plan.row_blocks;
  plan.blocks = units > most / steps ? most : units * steps;
  plan.ws_bytes = kTicketRegionBytes + (size_t)(plan.blocks * 2 * 8 * plan.tiles) * (a.D + 2) * sizeof(float);
  return plan;
}

int launch_paged_u4(const PagedArgs& a, const U4Plan& plan, void* ws, cudaStream_t s, const U4Some* some) {
  const int64_t rows = a.Hq / a.Hkv * a.L, keys = a.max_pages * a.page_size;
  // steps are counted in 32 bits: a launch takes as many row blocks and then requests as fit
  const int64_t unit = (keys + kStep - 1) / kStep + 1 + kUnitCost;
  const int64_t slice = std::min(plan.row_blocks, INT32_MAX / 2 / (a.Hkv * unit));
  if (keys > INT32_MAX - 4096 || rows > INT32_MAX / 2 || slice < 1)
    return fail(NVM_ERR_UNSUPPORTED, "paged_attention: 4-bit pages: too many rows or keys");
  const int64_t line = a.Hkv * slice * unit;
  U4Params p{};
  p.kp = static_cast<const uint8_t*>(a.k_pages);
  p.vp = static_cast<const uint8_t*>(a.v_pages);
  p.ks = static_cast<const uint8_t*>(a.k_scales);
  p.vs = static_cast<const uint8_t*>(a.v_scales);
  p.q_dtype = a.q_dtype;
  p.out_dtype = a.out_dtype;
  p.causal = a.is_causal;
  p.q_fast = a.q_dtype != NVM_F32 && (uintptr_t)a.q % 16 == 0;
  p.Hkv = (int)a.Hkv;
  p.L = (int)a.L;
  p.rows = (int)rows;
  p.P = (int)a.P;
  p.ps = (int)a.page_size;
  p.mp = a.P > 0 ? (int)a.max_pages : 0;  // a pool without pages: no key, and nothing to read
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.by_ps = FastDiv(a.page_size);
  p.tickets = static_cast<int*>(ws);
  p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kTicketRegionBytes);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + plan.blocks * 2 * 8 * plan.tiles * a.D);
  const int64_t part = std::min<int64_t>(INT32_MAX / line, INT32_MAX / 64);
  for (int64_t b0 = 0; b0 < a.B; b0 += part) {
    const int64_t first_row = b0 * a.Hq * a.L * a.D;
    p.B = (int)std::min(part, a.B - b0);
    p.q = static_cast<const uint8_t*>(a.q) + first_row * (int64_t)dtype_size(a.q_dtype);
    p.out = static_cast<uint8_t*>(a.out) + first_row * (int64_t)dtype_size(a.out_dtype);
    p.block_table = a.block_table + b0 * a.max_pages;
    p.context_lens = a.context_lens + b0;
    if (some != nullptr)
      p.some = U4Some{some->first + b0 * a.Hkv, some->rows + b0 * a.Hq * a.L, some->some + b0};
    for (int64_t r0 = 0; r0 < plan.row_blocks; r0 += slice) {
      p.row_block0 = (int)r0;
      p.row_blocks = (int)std::min(slice, plan.row_blocks - r0);
      const int st = a.scale_dtype == NVM_BF16 ? launch_d<__nv_bfloat16>(p, a.D, plan.tiles, plan.blocks, s)
                                               : launch_d<__half>(p, a.D, plan.tiles, plan.blocks, s);
      if (st != NVM_OK) return st;
    }
  }
  return NVM_OK;
}

}  // namespace nvm
