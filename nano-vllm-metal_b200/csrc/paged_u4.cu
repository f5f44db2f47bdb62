// paged_u4.cu -- paged attention over a cache held in 4 bits (u4.cuh has the row format).
//
// Semantics are those of the other paged kernels: positions at or past min(ctx, max_pages * page_size),
// holes (page id < 0 or >= P) and, with the causal limit, keys after l + ctx - L are skipped; a row that
// sees nothing is zero, and a key that no row sees has no influence whatever it holds.
//
// Mathematics.  With K = s c + z and V = s' c' + z' (one pair a group of 64 elements) a score is
//   q.k = sum over groups of s (q . c) + z (sum of q),
// and an output element of group g is (sum p s'_g c' + sum p z'_g) / sum p: codes enter the matrix
// instructions as they are, scales and offsets act on scores and weights.  A code becomes the f16 number
// 64 + code by one shift and one logic operation for two (bits 4-7 of 64.0h); the 64 is taken out again
// with sum q, and with the sum of the weights as the matrix unit saw them (a product with ones).
// Queries are held in f16, each row scaled by a power of two (exact for 16-bit queries).
//
// Weights are 2^(t - M), t the base-2 score and M a running reference per row, held in f16 once they
// are multiplied by s'.  M is kept within 2^10 of the largest t + log2 |v| so far, the largest
// contribution rather than the largest weight: f16 then holds what matters to 11 bits however small
// the values of the keys that are attended to.  Sums of weights and of p z' are fp32.
#include <algorithm>

#include "nvm_internal.h"
#include "u4.cuh"

namespace nvm {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;    // keys of a stage, one page lookup a lane
constexpr int kStages = 3;   // of each warp's own ring
constexpr float kSlack = 10.0f;    // log2 of how far a contribution may pass M
constexpr float kLeast = -40.0f;   // log2 of the least size that a key's values count as
constexpr float kNoKeys = -1e30f;  // M of a row that has seen no key

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
  float2* part_ml;  // [units][n_chunks][rows of a block]: (M, sum of weights)
  float* part_o;    // [units][n_chunks][rows of a block][D]
  int* tickets;     // [units], zero between calls
  int q_dtype, out_dtype, causal;
  int Hkv, L, rows, row_blocks, P, ps, mp, n_units, n_chunks, chunk;
  uint32_t ps_mul, ps_shift;  // key / ps = key * ps_mul >> ps_shift
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(there ? kBytes : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}
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
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// bits 4-7 of both halves as 64 + code
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(d) : "r"(w));
  return d;
}

// A tile's key in row m of a matrix fragment (and + 8 in row m + 8).  With the 16-byte parts of a
// row's 64 swapped by swizzle(), both the 8-byte reads of K (rows 2i, 2i + 1 and four lanes a row)
// and the 4-byte reads of V (rows 2c over the lanes c) touch every bank once.
__device__ __forceinline__ int key_of(int m) {
  const int base = (m >> 1 & 1) << 1 | m >> 2;
  return m & 1 ? (base ^ 1) + 4 : base;
}
__device__ __forceinline__ int swizzle(int key) { return (key >> 1 & 1) << 1; }

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
  // log2 of the largest number that the key's values may have
  __device__ __forceinline__ float size_log2() const {
    float m = fmaxf(fabsf(z[0]), 16.0f * s[0]);
    if constexpr (kGroups == 2) m = fmaxf(m, fmaxf(fabsf(z[1]), 16.0f * s[1]));
    return fmaxf(lg2(m), kLeast);
  }
};

// One block: kTiles x 8 query rows of one (request, kv head) against one chunk of keys, every warp
// on tiles of 32 keys of its own, joined in shared memory; chunks are joined by the unit's last block.
template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kWarps * 32, kTiles == 1 ? 4 : 3) paged_u4_kernel(const U4Params p) {
  using R = Ring<D>;
  constexpr int G = R::kGroups, kRows = 8 * kTiles;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_ml[kWarps][kRows];
  __shared__ uint32_t s_there[kWarps][kStages];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;

  const int chunk = blockIdx.x / p.n_units, unit = blockIdx.x - chunk * p.n_units;
  const int rb = unit % p.row_blocks, bh = unit / p.row_blocks, b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  const int row0 = rb * kRows, rows = min(kRows, p.rows - row0);
  const int ctx = p.context_lens[b];
  const int cap = p.mp * p.ps, limit = min(ctx, cap);
  // keys that the block's rows see: [0, most) by some row, [0, least) by every row
  int most = limit, least = limit;
  if (p.causal) {
    int lo = p.L, hi = 0;
    if (rows >= p.L) {
      lo = 0;
      hi = p.L - 1;
    } else {
      lo = row0 % p.L;
      hi = (row0 + rows - 1) % p.L;
      if (lo > hi) {
        lo = 0;
        hi = p.L - 1;
      }
    }
    most = min(limit, hi + ctx - p.L + 1);
    least = min(limit, lo + ctx - p.L + 1);
  }
  most = max(most, 0);
  // this unit's chunks: as many of p.chunk keys as it needs, evened out
  const int chunks = max(1, (most + p.chunk - 1) / p.chunk);
  if (chunk >= chunks) return;
  const int share = ((most + chunks - 1) / chunks + kWarps * kTile - 1) / (kWarps * kTile) * (kWarps * kTile);
  const int begin = min(chunk * share, most), end = min(begin + share, most);

  const size_t out_row0 = (size_t)bh * p.rows + row0;
  uint8_t* ring = smem + warp * R::kWarp;
  const uint32_t ring_at = smem_u32(ring);
  const int32_t* bt = p.block_table + (size_t)b * p.mp;

  auto page_of_key = [&](int key) -> int {
    if (key >= end) return -1;
    const int pid = __ldg(bt + (uint32_t)((uint64_t)(uint32_t)key * p.ps_mul >> p.ps_shift));
    return pid < p.P ? pid : -1;
  };
  // copies the tile whose first key is k0 (a lane's key lies in page pid) into a stage
  auto issue = [&](int k0, int pid, int stage) {
    const uint32_t page = (uint32_t)((uint64_t)(uint32_t)(k0 + lane) * p.ps_mul >> p.ps_shift);
    const uint32_t off = (uint32_t)(k0 + lane) - page * (uint32_t)p.ps;
    const uint32_t row = pid < 0 ? 0xffffffffu : ((uint32_t)pid * p.Hkv + kvh) * p.ps + off;
    const uint32_t there = __ballot_sync(0xffffffffu, pid >= 0);
    if (lane == 0) s_there[warp][stage] = there;
    const uint32_t at = ring_at + stage * R::kStage;
    constexpr int kParts = R::kRow / 16, kKeysAStep = 32 / kParts;
#pragma unroll
    for (int i = 0; i < kTile / kKeysAStep; ++i) {
      const int key = i * kKeysAStep + lane / kParts, part = lane % kParts;
      const uint32_t krow = __shfl_sync(0xffffffffu, row, key);
      const bool ok = krow != 0xffffffffu;
      const size_t src = ok ? (size_t)krow * R::kRow + part * 16 : 0;
      const uint32_t dst = at + key * R::kRow + ((D == 128 ? part ^ swizzle(key) : part) << 4);
      cp_async16(dst, p.kp + src, ok);
      cp_async16(dst + R::kV, p.vp + src, ok);
    }
    const size_t src = pid >= 0 ? (size_t)row * (4 * G) : 0;
    cp_async_small<4 * G>(at + R::kKs + lane * 4 * G, p.ks + src, pid >= 0);
    cp_async_small<4 * G>(at + R::kVs + lane * 4 * G, p.vs + src, pid >= 0);
  };

  const int step = kWarps * kTile;
  int k_next = begin + warp * kTile;  // first key of the tile to copy next
  int pid = page_of_key(k_next + lane);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (k_next < end) issue(k_next, pid, s);
    cp_async_commit();
    k_next += step;
    pid = page_of_key(k_next + lane);
  }

  // Queries as B fragments (lane: row r of each tile of 8, 16 elements a group), scaled per row so that
  // the largest is in [2^8, 2^9); kap undoes it and turns scores to base 2.
  uint32_t qf[kTiles][G][4][2];
  float kap[kTiles][2], qsum[kTiles][2][G];
  int seen[kTiles][2];  // keys [0, seen) are seen by the lane's rows 2c, 2c + 1
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    float x[G][16], top = 0.0f;
    const int row = 8 * j + r;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float2 v = make_float2(0.0f, 0.0f);
        if (row < rows) {
          const int64_t at = (int64_t)(out_row0 + row) * D + g * kU4Group + c * 16 + e;
          v = p.q_dtype == NVM_BF16  ? load_pair<__nv_bfloat16>(p.q, at)
              : p.q_dtype == NVM_F16 ? load_pair<__half>(p.q, at)
                                     : load_pair<float>(p.q, at);
        }
        x[g][e] = v.x;
        x[g][e + 1] = v.y;
        top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e2 = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 100);
    float up = __uint_as_float((uint32_t)(127 + 8 - e2) << 23);
    float down = p.scale_log2 * __uint_as_float((uint32_t)(127 - 8 + e2) << 23);
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
            const __half2 v = __floats2half2_rn(x[g][8 * w + 2 * h + i] * up, x[g][8 * w + 2 * h + i + 4] * up);
            qf[j][g][2 * w + h][i] = *reinterpret_cast<const uint32_t*>(&v);
            const float2 f = __half22float2(v);
            sum[g] += f.x + f.y;
          }
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kap[j][i] = __shfl_sync(0xffffffffu, down, (2 * c + i) * 4);
#pragma unroll
      for (int g = 0; g < G; ++g) qsum[j][i][g] = __shfl_sync(0xffffffffu, sum[g], (2 * c + i) * 4);
      const int rr = row0 + 8 * j + 2 * c + i;
      seen[j][i] = rr - row0 >= rows ? INT32_MAX : p.causal ? min(limit, rr % p.L + ctx - p.L + 1) : limit;
    }
  }

  float acc[G][4][kTiles][4], wsum[G][kTiles][4], M[kTiles][2], l[kTiles][2], zsum[kTiles][2][G];
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
    }
    M[j][0] = M[j][1] = kNoKeys;
    l[j][0] = l[j][1] = 0.0f;
  }

  const int kr = key_of(r), kc0 = key_of(2 * c), kc1 = key_of(2 * c + 1);
  // byte offsets inside a stage: K rows of fragment row r, V rows of fragment columns 2c and 2c + 1
  uint32_t k_off[G], v_off0[G], v_off1[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if constexpr (D == 128) {
      k_off[g] = kr * R::kRow + (((2 * g + (c >> 1)) ^ swizzle(kr)) << 4) + (c & 1) * 8;
      v_off0[g] = R::kV + kc0 * R::kRow + (((2 * g + (r >> 2)) ^ swizzle(kc0)) << 4) + (r & 3) * 4;
      v_off1[g] = R::kV + kc1 * R::kRow + (((2 * g + (r >> 2)) ^ swizzle(kc1)) << 4) + (r & 3) * 4;
    } else {
      k_off[g] = kr * R::kRow + c * 8;
      v_off0[g] = R::kV + kc0 * R::kRow + r * 4;
      v_off1[g] = R::kV + kc1 * R::kRow + r * 4;
    }
  }

  int stage = 0, stage_in = kStages - 1;
  for (int k0 = begin + warp * kTile; k0 < end; k0 += step) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    if (k_next < end) issue(k_next, pid, stage_in);
    cp_async_commit();
    k_next += step;
    pid = page_of_key(k_next + lane);
    const uint32_t at = ring_at + stage * R::kStage;
    const uint32_t there = s_there[warp][stage];
    stage_in = stage;
    stage = stage + 1 == kStages ? 0 : stage + 1;

    // x[mt][j][e]: score / kap of key key_of(r) + 16 mt + 8 (e / 2), row 2c + e % 2 of tile j
    float x[2][kTiles][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      Pairs<T, G> a, d;
      a.load(at + R::kKs + (kr + 16 * mt) * 4 * G);
      d.load(at + R::kKs + (kr + 16 * mt + 8) * 4 * G);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint2 lo = lds64(at + k_off[g] + 16 * mt * R::kRow), hi = lds64(at + k_off[g] + (16 * mt + 8) * R::kRow);
        float dot[kTiles][4];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) dot[j][0] = dot[j][1] = dot[j][2] = dot[j][3] = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t u = w == 0 ? lo.x : lo.y, v = w == 0 ? hi.x : hi.y;
          const uint32_t a0[4] = {codes_f16(u << 4), codes_f16(v << 4), codes_f16(u), codes_f16(v)};
          const uint32_t a1[4] = {codes_f16(u >> 4), codes_f16(v >> 4), codes_f16(u >> 8), codes_f16(v >> 8)};
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            mma16816<__half>(dot[j], a0, qf[j][g][2 * w][0], qf[j][g][2 * w][1]);
            mma16816<__half>(dot[j], a1, qf[j][g][2 * w + 1][0], qf[j][g][2 * w + 1][1]);
          }
        }
        const float za = fmaf(-64.0f, a.s[g], a.z[g]), zd = fmaf(-64.0f, d.s[g], d.z[g]);
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = e < 2 ? a.s[g] : d.s[g], z = e < 2 ? za : zd;
            const float off = g == 0 ? z * qsum[j][e & 1][g] : fmaf(z, qsum[j][e & 1][g], x[mt][j][e]);
            x[mt][j][e] = fmaf(s, dot[j][e], off);
          }
      }
    }

    Pairs<T, G> vz[2][2];
    float size[2][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        vz[mt][h].load(at + R::kVs + (kr + 16 * mt + 8 * h) * 4 * G);
        size[mt][h] = vz[mt][h].size_log2();
      }

    const bool masked = there != 0xffffffffu || k0 + kTile > least;
    if (masked) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = kr + 16 * mt + 8 * (e >> 1);
            const bool ok = (there >> key & 1) && k0 + key < seen[j][e & 1];
            if (!ok) x[mt][j][e] = kap[j][e & 1] < 0.0f ? INFINITY : -INFINITY;  // kap * x = -inf
          }
    }

    // references that some contribution passes by 2^kSlack move to the largest one
    float u[2][kTiles][4];
    bool over = false;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[mt][j][e] = fmaf(kap[j][e & 1], x[mt][j][e], -M[j][e & 1]);
          over |= u[mt][j][e] + size[mt][e >> 1] > kSlack;
        }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = M[j][i];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaf(kap[j][i], x[mt][j][2 * h + i], size[mt][h]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float fade = ex2(M[j][i] - top);
          M[j][i] = top;
          l[j][i] *= fade;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            zsum[j][i][g] *= fade;
            wsum[g][j][i] *= fade;
            wsum[g][j][2 + i] *= fade;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              acc[g][t][j][i] *= fade;
              acc[g][t][j][2 + i] *= fade;
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) u[mt][j][2 * h + i] = fmaf(kap[j][i], x[mt][j][2 * h + i], -top);
        }
    }

    // weights, their sums, and the weights times the values' scales as B fragments
    uint32_t pf[2][kTiles][G][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Pairs<T, G>& v = vz[mt][h];
          const float w0 = ex2(u[mt][j][2 * h]), w1 = ex2(u[mt][j][2 * h + 1]);
          l[j][0] += w0;
          l[j][1] += w1;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float s0 = w0 * v.s[g], s1 = w1 * v.s[g], z0 = w0 * v.z[g], z1 = w1 * v.z[g];
            if (masked) {  // a key that the row does not see counts nothing, whatever its values
              if (w0 == 0.0f) s0 = z0 = 0.0f;
              if (w1 == 0.0f) s1 = z1 = 0.0f;
            }
            zsum[j][0][g] += z0;
            zsum[j][1][g] += z1;
            pf[mt][j][g][h] = transpose8x8(pack2<__half>(s0, s1));
          }
        }

    const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t k00 = lds32(at + v_off0[g] + 16 * mt * R::kRow), k01 = lds32(at + v_off1[g] + 16 * mt * R::kRow);
        const uint32_t k80 = lds32(at + v_off0[g] + (16 * mt + 8) * R::kRow), k81 = lds32(at + v_off1[g] + (16 * mt + 8) * R::kRow);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          const uint32_t y = prmt(k00, k01, sel), y8 = prmt(k80, k81, sel);
          const uint32_t a0[4] = {codes_f16(y << 4), codes_f16(y), codes_f16(y8 << 4), codes_f16(y8)};
          const uint32_t a1[4] = {codes_f16(y >> 4), codes_f16(y >> 8), codes_f16(y8 >> 4), codes_f16(y8 >> 8)};
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            mma16816<__half>(acc[g][2 * half][j], a0, pf[mt][j][g][0], pf[mt][j][g][1]);
            mma16816<__half>(acc[g][2 * half + 1][j], a1, pf[mt][j][g][0], pf[mt][j][g][1]);
          }
        }
#pragma unroll
        for (int j = 0; j < kTiles; ++j) mma16816<__half>(wsum[g][j], one, pf[mt][j][g][0], pf[mt][j][g][1]);
      }
  }
  cp_async_wait<0>();

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
      if (r == 0) s_ml[warp][row] = make_float2(M[j][i], l[j][i]);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float more = fmaf(-64.0f, wsum[g][j][i], zsum[j][i][g]);
        float* dst = part + row * kPitch + g * kU4Group + r * 8;
#pragma unroll
        for (int t = 0; t < 4; t += 2)
          *reinterpret_cast<float4*>(dst + 2 * t) = make_float4(acc[g][t][j][i] + more, acc[g][t][j][2 + i] + more,
                                                                acc[g][t + 1][j][i] + more, acc[g][t + 1][j][2 + i] + more);
      }
    }
  __syncthreads();

  const size_t slot = ((size_t)unit * p.n_chunks + chunk) * kRows;
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
    if (chunks == 1) {
      store_dyn(p.out, (int64_t)(out_row0 + row) * D + d, p.out_dtype, sum == 0.0f ? 0.0f : o / sum);
    } else {
      p.part_o[(slot + row) * D + d] = o;
      if (d == 0) p.part_ml[slot + row] = make_float2(top, sum);
    }
  }
  if (chunks == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.tickets + unit, 1) == chunks - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (threadIdx.x == 0) p.tickets[unit] = 0;
  const size_t base = (size_t)unit * p.n_chunks * kRows;
  for (int i = threadIdx.x; i < rows * D; i += kWarps * 32) {
    const int row = i / D, d = i - row * D;
    float top = kNoKeys, sum = 0.0f, o = 0.0f;
    for (int k = 0; k < chunks; ++k) top = fmaxf(top, __ldcg(&p.part_ml[base + (size_t)k * kRows + row].x));
    for (int k = 0; k < chunks; ++k) {
      const float2 ml = __ldcg(&p.part_ml[base + (size_t)k * kRows + row]);
      const float f = ex2(ml.x - top);
      sum = fmaf(f, ml.y, sum);
      o = fmaf(f, __ldcg(&p.part_o[(base + (size_t)k * kRows + row) * D + d]), o);
    }
    store_dyn(p.out, (int64_t)(out_row0 + row) * D + d, p.out_dtype, sum == 0.0f ? 0.0f : o / sum);
  }
}

template <typename T, int D, int kTiles>
int launch(const U4Params& p, int64_t blocks, cudaStream_t s) {
  constexpr int bytes = kWarps * Ring<D>::kWarp;
  const cudaError_t e = cudaFuncSetAttribute(paged_u4_kernel<T, D, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return check_cuda(e, "paged_attention: cudaFuncSetAttribute");
  paged_u4_kernel<T, D, kTiles><<<(unsigned)blocks, kWarps * 32, bytes, s>>>(p);
  return check_cuda(cudaGetLastError(), "paged_attention: 4-bit kernel launch");
}

template <typename T>
int launch_d(const U4Params& p, int64_t D, int tiles, int64_t blocks, cudaStream_t s) {
  if (D == 128) return tiles == 1 ? launch<T, 128, 1>(p, blocks, s) : launch<T, 128, 2>(p, blocks, s);
  return tiles == 1 ? launch<T, 64, 1>(p, blocks, s) : launch<T, 64, 2>(p, blocks, s);
}

}  // namespace

U4Plan plan_paged_u4(const PagedArgs& a) {
  U4Plan plan{};
  const int64_t rows = a.Hq / a.Hkv * a.L, keys = a.max_pages * a.page_size;
  plan.tiles = rows <= 8 ? 1 : 2;
  plan.row_blocks = (rows + 8 * plan.tiles - 1) / (8 * plan.tiles);
  plan.units = a.B * a.Hkv * plan.row_blocks;
  const int64_t slots = 148 * 4, least = kWarps * kTile;
  int64_t chunk = (keys * plan.units + 3 * slots - 1) / (3 * slots);
  chunk = std::max<int64_t>((chunk + least - 1) / least * least, least);
  if (plan.units > (int64_t)(kTicketRegionBytes / sizeof(int))) chunk = std::max<int64_t>(keys, 1);
  plan.chunk = chunk;
  plan.n_chunks = std::max<int64_t>((keys + chunk - 1) / chunk, 1);
  if (plan.n_chunks > 1)
    plan.ws_bytes = kTicketRegionBytes + (size_t)(plan.units * plan.n_chunks * 8 * plan.tiles) * (a.D + 2) * sizeof(float);
  return plan;
}

int launch_paged_u4(const PagedArgs& a, const U4Plan& plan, void* ws, cudaStream_t s) {
  const int64_t blocks = plan.units * plan.n_chunks;
  if (blocks > INT32_MAX || a.max_pages * a.page_size > INT32_MAX - 4096 || a.Hq / a.Hkv * a.L > INT32_MAX / 2)
    return fail(NVM_ERR_UNSUPPORTED, "paged_attention: 4-bit pages: too many rows or keys");
  U4Params p{};
  p.q = a.q;
  p.kp = static_cast<const uint8_t*>(a.k_pages);
  p.vp = static_cast<const uint8_t*>(a.v_pages);
  p.ks = static_cast<const uint8_t*>(a.k_scales);
  p.vs = static_cast<const uint8_t*>(a.v_scales);
  p.block_table = a.block_table;
  p.context_lens = a.context_lens;
  p.out = a.out;
  p.q_dtype = a.q_dtype;
  p.out_dtype = a.out_dtype;
  p.causal = a.is_causal;
  p.Hkv = (int)a.Hkv;
  p.L = (int)a.L;
  p.rows = (int)(a.Hq / a.Hkv * a.L);
  p.row_blocks = (int)plan.row_blocks;
  p.P = (int)a.P;
  p.ps = (int)a.page_size;
  p.mp = (int)a.max_pages;
  p.n_units = (int)plan.units;
  p.n_chunks = (int)plan.n_chunks;
  p.chunk = (int)std::min<int64_t>(plan.chunk, INT32_MAX / 2);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  // key / ps for keys below 2^31: with 2^(n - 1) < ps <= 2^n and m = floor(2^(31 + n) / ps) + 1 the error
  // m ps - 2^(31 + n) is at most 2^n, so key * m >> 31 + n is exact
  int n = 0;
  while ((int64_t(1) << n) < a.page_size) ++n;
  p.ps_mul = (uint32_t)((uint64_t(1) << (31 + n)) / (uint64_t)a.page_size + 1);
  p.ps_shift = (uint32_t)(31 + n);
  if (plan.ws_bytes > 0) {
    p.tickets = static_cast<int*>(ws);
    p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kTicketRegionBytes);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + plan.units * plan.n_chunks * 8 * plan.tiles * a.D);
  }
  return a.scale_dtype == NVM_BF16 ? launch_d<__nv_bfloat16>(p, a.D, plan.tiles, blocks, s)
                                   : launch_d<__half>(p, a.D, plan.tiles, blocks, s);
}

}  // namespace nvm
