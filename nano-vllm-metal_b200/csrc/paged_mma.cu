// paged_mma.cu -- plan and dispatch of the tensor-core paged attention kernel
// (paged_mma.cuh): kernel variants per shape class, split-K sizing, cluster merges.
#include "paged_mma.cuh"

namespace nvm {
namespace {

constexpr int kDefaultDecodeVariant = 3;
constexpr int kDefaultN8Variant = 7;  // c4 int8 prefers 4 (2 warps, 8 stages) by 1%
constexpr int kDefaultM3Variant = 1;
// longest chunk (16-key tiles) the one-wave sizing of the n8 tile hands a CTA
constexpr int64_t kOneWaveTiles = 128;

// CTAs of one n8 kernel instance resident on an SM (registers and shared memory), asked
// of the runtime once; without a device (workspace sizing on a host) the shared-memory
// bound, at most 8 (the register bound of the instances built here: <= 128 a thread).
template <typename KvT, typename ScaleT, int D, int NWK, int NS_>
int n8_resident() {
  using C = Cfg<KvT, D, 0, NWK, NS_>;
  static std::atomic<int> cached{0};
  int n = cached.load(std::memory_order_relaxed);
  if (n > 0) return n;
  n = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ensure_smem_attr<KvT, ScaleT, D, 0, NWK, NS_, false>() != NVM_OK ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_mma_kernel<KvT, ScaleT, D, 0, NWK, NS_, false>, C::kThreads,
                                                    C::kSmemBytes) != cudaSuccess ||
      n <= 0) {
    cudaGetLastError();
    n = 233472 / (C::kSmemBytes + 1024);
    n = n < 1 ? 1 : (n > 8 ? 8 : n);
    return n;  // not cached: a later call with a device asks the runtime
  }
  cached.store(n, std::memory_order_relaxed);
  return n;
}

template <typename KvT, typename ScaleT, int D>
int n8_resident_variant(int variant) {
  switch (variant) {  // the (NWK, NS) of each variant, as launch_decode maps them
    case 0: return n8_resident<KvT, ScaleT, D, 4, 0>();
    case 1: return n8_resident<KvT, ScaleT, D, 4, 12>();
    case 2: return n8_resident<KvT, ScaleT, D, 2, 2>();
    case 4: return n8_resident<KvT, ScaleT, D, 2, 8>();
    case 5: return n8_resident<KvT, ScaleT, D, 4, 4>();
    case 6: return n8_resident<KvT, ScaleT, D, 1, 4>();
    case 7: return n8_resident<KvT, ScaleT, D, 2, 4>();
    case 8: return n8_resident<KvT, ScaleT, D, 1, 6>();
    default: return n8_resident<KvT, ScaleT, D, 2, 6>();
  }
}

int n8_resident_per_sm(const PagedArgs& a, int variant) {
  if (a.kv_dtype == NVM_I8) return n8_resident_variant<int8_t, __half, 128>(variant);
  if (a.kv_dtype == NVM_F16)
    return a.D == 64 ? n8_resident_variant<__half, __half, 64>(variant) : n8_resident_variant<__half, __half, 128>(variant);
  return a.D == 64 ? n8_resident_variant<__nv_bfloat16, __nv_bfloat16, 64>(variant)
                   : n8_resident_variant<__nv_bfloat16, __nv_bfloat16, 128>(variant);
}

int sm_count_cached() {
  static std::atomic<int> cached{0};
  int n = cached.load(std::memory_order_relaxed);
  if (n > 0) return n;
  int dev = 0;
  n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      n <= 0) {
    cudaGetLastError();
    return 148;
  }
  cached.store(n, std::memory_order_relaxed);
  return n;
}

// Kernel variants (consumer warps along keys NWK, stage depth NS) per shape class.
// Fewer warps and stages per CTA let more CTAs -- and more independent TMA
// producers -- share an SM, which keeps more page loads in flight: on B200 the
// 16-bit decode reached 98% of measured HBM bandwidth with 2 consumer warps and 6
// stages (4 CTAs per SM) against 64% with 4 warps and 8 stages (2 CTAs per SM).
// NVM_ATTN_DECODE_CFG selects another variant (for sweeps).
template <typename KvT, typename ScaleT, int D, int NWM>
int launch_decode(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  switch (plan.variant) {
    case 0: return launch_cfg<KvT, ScaleT, D, NWM, 4>(a, plan, ws, s);
    case 1: return launch_cfg<KvT, ScaleT, D, NWM, 4, 12>(a, plan, ws, s);
    case 2: return launch_cfg<KvT, ScaleT, D, NWM, 2, 2>(a, plan, ws, s);
    case 3: return launch_cfg<KvT, ScaleT, D, NWM, 2, 6>(a, plan, ws, s);
    case 4: return launch_cfg<KvT, ScaleT, D, NWM, 2, 8>(a, plan, ws, s);
    case 5: return launch_cfg<KvT, ScaleT, D, NWM, 4, 4>(a, plan, ws, s);
    case 6: return launch_cfg<KvT, ScaleT, D, NWM, 1, 4>(a, plan, ws, s);
    case 7: return launch_cfg<KvT, ScaleT, D, NWM, 2, 4>(a, plan, ws, s);
    case 8: return launch_cfg<KvT, ScaleT, D, NWM, 1, 6>(a, plan, ws, s);
    default: return launch_cfg<KvT, ScaleT, D, NWM, 2, 6>(a, plan, ws, s);
  }
}

// Three 16-row m-tiles (e.g. 8 q heads x 5 verify tokens = 40 rows).
template <typename KvT, typename ScaleT, int D>
int launch_m3(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  switch (plan.variant) {
    case 0: return launch_cfg<KvT, ScaleT, D, 3, 2>(a, plan, ws, s);
    case 1: return launch_cfg<KvT, ScaleT, D, 3, 1, 4>(a, plan, ws, s);
    case 2: return launch_cfg<KvT, ScaleT, D, 3, 1, 6>(a, plan, ws, s);
    case 3: return launch_cfg<KvT, ScaleT, D, 3, 2, 6>(a, plan, ws, s);
    default: return launch_cfg<KvT, ScaleT, D, 3, 1, 4>(a, plan, ws, s);
  }
}

template <typename KvT, typename ScaleT, int D>
int launch_d(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  switch (plan.nwm) {
    case 0: return launch_decode<KvT, ScaleT, D, 0>(a, plan, ws, s);
    case 1: return launch_decode<KvT, ScaleT, D, 1>(a, plan, ws, s);
    case 2: return launch_cfg<KvT, ScaleT, D, 2, 2>(a, plan, ws, s);
    case 3: return launch_m3<KvT, ScaleT, D>(a, plan, ws, s);
    default: return launch_cfg<KvT, ScaleT, D, 4, 1>(a, plan, ws, s);
  }
}

}  // namespace

MmaPlan plan_paged_mma(const PagedArgs& a) {
  MmaPlan plan{};
  plan.eligible = false;
  const bool kv16 = a.kv_dtype == NVM_F16 || a.kv_dtype == NVM_BF16;
  const bool kv8 = a.kv_dtype == NVM_I8 && a.D == 128 && (a.scale_dtype == NVM_F16 || a.scale_dtype == NVM_BF16);
  if (!(kv16 && (a.D == 64 || a.D == 128)) && !kv8) return plan;
  const bool dense = a.dense != 0;
  if (dense ? a.page_size < 16 : (a.page_size % 16) != 0) return plan;
  if (a.P <= 0 || a.P > INT32_MAX || a.Hkv > INT32_MAX || a.page_size > INT32_MAX) return plan;
  if (a.max_pages <= 0) return plan;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a.k_pages) || !al16(a.v_pages)) return plan;
  // q is read as element pairs
  if ((reinterpret_cast<uintptr_t>(a.q) & (a.q_dtype == NVM_F32 ? 7 : 3)) != 0) return plan;
  if (kv8 && (!al16(a.k_scales) || !al16(a.v_scales))) return plan;
  const int64_t M = (a.Hq / a.Hkv) * a.L;
  plan.nwm = M <= 16 ? 1 : (M <= 32 ? 2 : (M <= 48 ? 3 : 4));
  // at most eight query rows per kv head: the n8 tile (nwm = 0)
  if (M <= 8 && env_int("NVM_ATTN_N8", 1) != 0) plan.nwm = 0;
  plan.nwk = plan.nwm <= 1 ? 4 : (plan.nwm == 4 ? 1 : 2);
  // variant -> consumer warps along keys (must match launch_decode / launch_m3)
  plan.variant = -1;
  if (plan.nwm <= 1) {
    static const int kWarps1[9] = {4, 4, 2, 2, 2, 4, 1, 2, 1};
    // the n8 tile runs without a producer warp: small CTAs with a short ring
    // (2 warps x 4 stages) let the most of them share an SM (one CTA per unit with a
    // producer and 12 consumer warps measured 1.9x slower on config 1: a unit's pages
    // have to come through many SMs)
    int dflt = plan.nwm == 0 ? kDefaultN8Variant : kDefaultDecodeVariant;
    // n8 tile, 16-bit pages, short contexts, more units than the default variant's CTA
    // slots but no more than those of 2 warps x 2 stages (8 CTAs per SM against 6): the
    // smaller ring runs the launch as one wave (B = 128 at 1-1.1K keys, 32/8 heads: 92 us
    // against 112 us).  Launches that need several waves either way keep the deeper ring
    // (B = 160 at 600-1000 keys, 16/8 heads: 101 us against 107 us with 2 x 2; config 3:
    // 2 x 4 stages 7249-7292 GB/s against 7090-7137).
    if (plan.nwm == 0 && kv16 && !dense && env_int("NVM_ATTN_WAVE_RULE", 1) != 0) {
      const int64_t units = a.B * a.Hkv, sms = sm_count_cached();
      int64_t tiles = (a.max_pages * a.page_size + 15) / 16;
      if (a.window > 0 && (a.sinks + 15) / 16 + (a.window + 15) / 16 + 1 < tiles)
        tiles = (a.sinks + 15) / 16 + (a.window + 15) / 16 + 1;
      if (tiles <= kOneWaveTiles && units > sms * n8_resident_per_sm(a, dflt) && units <= sms * n8_resident_per_sm(a, 2))
        dflt = 2;
    }
    plan.variant = (int)env_int("NVM_ATTN_DECODE_CFG", dflt);
    if (plan.variant < 0 || plan.variant > 8) plan.variant = 3;
    if (paged_is_ext(a)) plan.variant = dflt;  // the windowed kernel is built for the defaults only
    plan.nwk = kWarps1[plan.variant];
  } else if (plan.nwm == 3) {
    static const int kWarps3[4] = {2, 1, 1, 2};
    plan.variant = (int)env_int("NVM_ATTN_M3_CFG", kDefaultM3Variant);
    if (plan.variant < 0 || plan.variant > 3) plan.variant = 1;
    if (paged_is_ext(a)) plan.variant = kDefaultM3Variant;
    plan.nwk = kWarps3[plan.variant];
  }
  plan.rows_per_block = plan.nwm == 0 ? 8 : 16 * plan.nwm;
  plan.n_row_blocks = (M + plan.rows_per_block - 1) / plan.rows_per_block;
  // Under a window a block of rows of one head reaches over that many keys more than the window;
  // one that spans two heads' ends would walk the windows of all L tokens.
  plan.head_blocks = 0;
  if (a.window > 0 && plan.nwm == 4 && a.L >= plan.rows_per_block) {
    plan.head_blocks = (a.L + plan.rows_per_block - 1) / plan.rows_per_block;
    plan.n_row_blocks = plan.head_blocks * (a.Hq / a.Hkv);
  }
  plan.rows_real = M < plan.rows_per_block ? M : plan.rows_per_block;
  plan.n_units = a.B * a.Hkv * plan.n_row_blocks;
  if (plan.n_units > INT32_MAX) return plan;
  const bool can_split = plan.n_units <= kMaxUnits;
  int64_t keys = a.max_pages * a.page_size;
  if (dense) keys = a.page_size;
  int64_t tiles_max = (keys + 15) / 16;
  const bool ext = paged_is_ext(a);
  bool even_units = false;  // a window cuts every unit to the same length
  // the windowed kernel counts keys and pool rows in 32 bits
  if (ext && (keys >= (int64_t(1) << 30) || a.P * a.Hkv * a.page_size > INT32_MAX - 64)) return plan;
  if (a.window > 0) {
    // the sinks' tiles and those that the windows of L tokens touch
    // (without the causal limit every row sees on to the last key)
    const int64_t span = a.is_causal && plan.head_blocks > 0 ? plan.rows_per_block : a.L;
    const int64_t seen = (a.sinks + 15) / 16 + (a.window + span - 1 + 15) / 16 + 1;
    if (seen < tiles_max) {
      tiles_max = seen;
      even_units = true;
    }
  }
  // the kernel's index arithmetic runs in 32 bits
  if (tiles_max >= INT32_MAX / 2 || M >= INT32_MAX) return plan;
  int64_t ct;
  if (dense || !can_split) {
    ct = tiles_max;  // dense callers pass no workspace: never split
  } else {
    // n8 tile: enough chunks for about six waves of its 8 CTAs per SM if every sequence
    // were as long as the longest: ragged contexts leave many chunks empty, and with
    // fewer waves the last one runs mostly idle (config 4, 64 sequences of 8K-32K keys:
    // 160-tile chunks 4777-4807 GB/s against 4533-4564 with 256; config 3 stays at the
    // 256 cap).  Multi-row tiles keep about 16 chunk CTAs per SM.
    const int64_t sms = sm_count_cached();
    const int64_t target = plan.nwm == 0 ? sms * 48 : sms * 16;
    ct = (plan.n_units * tiles_max + target - 1) / target;
    ct = ((ct + 15) / 16) * 16;
    if (ct < 16) ct = 16;
    if (ct > kMaxChunkTiles) ct = kMaxChunkTiles;
    // Short contexts (the n8 tile): many 16-tile chunks cost more in per-CTA set-up,
    // merges and partial waves than they gain in balance.  When the units fit in the
    // CTA slots the SMs hold at once, each is cut into the fewest equal chunks that give
    // about four CTAs per SM (enough page loads in flight to keep HBM busy), within one
    // wave, if those chunks are at most kOneWaveTiles long: B = 64 at 1-1.1K keys (32/8
    // heads) one 70-tile chunk a unit, 50.5 us against 65.5 us with five 14-tile chunks;
    // B = 32 at 2K keys three 44-tile chunks, 53 us against 66 us.  Otherwise chunks are
    // at least 48 tiles long (B = 128 at 1-1.1K keys: 2 x 35 tiles, 105 us against
    // 121 us; B = 256 at 512 keys: one 36-tile chunk, 104 us against 132 us).
    // NVM_ATTN_WAVE_RULE=0 keeps the six-wave sizing alone (sweeps).
    if (plan.nwm == 0 && env_int("NVM_ATTN_WAVE_RULE", 1) != 0) {
      const int64_t slots = sms * n8_resident_per_sm(a, plan.variant);
      bool one_wave = false;
      if (plan.n_units <= slots) {
        int64_t nc = (4 * sms + plan.n_units - 1) / plan.n_units;
        const int64_t nc_max = slots / plan.n_units;
        if (nc > nc_max) nc = nc_max;
        if (nc < 1) nc = 1;
        int64_t ct1 = (tiles_max + nc - 1) / nc;
        // Windowed / scored calls with few units: up to eight chunks, one cluster, down to four
        // tiles each (8 units of 35 tiles: seven chunks of 5 against three of 16).
        const int64_t least = ext && tiles_max <= 128 ? (tiles_max > 32 ? (tiles_max + 7) / 8 : 4) : 16;
        if (ct1 < least) ct1 = least;
        if (ct1 <= kOneWaveTiles) {
          ct = ct1;
          one_wave = true;
        }
      }
      if (!one_wave) {
        int64_t floor_ct = tiles_max < 48 ? tiles_max : 48;
        // Long contexts (>= 16K keys) with units enough for two waves of 128-tile chunks:
        // chunks of at least 128 tiles (one rank's kv-head shard of config 3 at 8 GPUs,
        // 256 units of 4K-32K keys: 380 us against 387 us with the six-wave 80 tiles;
        // config 4's 160 and config 3's 256 are above the floor anyway).
        if (tiles_max >= 1024 && plan.n_units * ((tiles_max + 127) / 128) >= 2 * slots) floor_ct = 128;
        if (ct < floor_ct) ct = floor_ct;
        // Units that a window makes equally long: the fewest chunks whose last wave is about
        // half full to nearly full (a last wave just begun costs the most).  Windows of 4096
        // keys, 8 kv heads, against the sizing above: 40 requests 118 / 133 us, 56: 158 / 174,
        // 64: 174 / 181, 100: 267 / 276, 128: 351 / 358; 48 and 80 within 2 % either way.
        for (int64_t nc = 2; even_units && nc <= 7; ++nc) {
          const int64_t part = (plan.n_units * nc) % slots;
          const int64_t ct1 = (tiles_max + nc - 1) / nc;
          if (ct1 <= kMaxChunkTiles && ct1 >= 16 && part * 20 >= slots * 9 && part * 20 <= slots * 19) {
            ct = ct1;
            break;
          }
        }
      }
    }
    // the longest context split evenly over that many chunks (B = 512 at 1024 tokens:
    // 2 x 32 tiles, 343 us, instead of 48 + 16, 391 us)
    if (ct < tiles_max) {
      const int64_t nc = (tiles_max + ct - 1) / ct;
      ct = (tiles_max + nc - 1) / nc;
    }
    const int64_t forced = env_int("NVM_ATTN_CHUNK_TILES", 0);
    if (forced > 0) ct = forced < kMaxChunkTiles ? forced : kMaxChunkTiles;
    if (ct > tiles_max) ct = tiles_max;
  }
  if (ct < 1) ct = 1;
  if (ct > kMaxChunkTiles && !dense) ct = kMaxChunkTiles;
  plan.chunk_tiles = ct;
  plan.n_chunks = (tiles_max + ct - 1) / ct;
  if (plan.n_chunks < 1) plan.n_chunks = 1;
  if (plan.n_chunks > 65535) return plan;
  if (!can_split && !dense && plan.n_chunks > 1) {
    // A chunk's page table holds kMaxChunkTiles tiles, so longer contexts are cut whatever the
    // number of units, but there are no tickets for so many: the caller takes the batch in parts.
    plan.max_batch = kMaxUnits / (a.Hkv * plan.n_row_blocks);
    return plan;
  }
  // n8 tile with 2..8 chunks: the chunks of a unit merge inside a thread-block cluster
  // (distributed shared memory) instead of through the workspace, which takes the
  // global-memory round trips of the split-K merge off every unit's critical path.
  // Every CTA of a cluster stays resident until its unit is merged, so chunks without
  // keys (ragged contexts) idle in their slots, and a cluster launches only when all
  // its CTAs fit at once; the cluster merge is therefore used when the launch fits in
  // one wave (B = 128 at 1-1.1K keys, 2 chunks over two waves: 125 us in clusters
  // against 105 us through the workspace).
  // NVM_ATTN_CLUSTER: 0 never, 2 whenever 2..8 chunks (sweeps), otherwise the rule above.
  plan.cluster = 0;
  const int64_t cl_mode = env_int("NVM_ATTN_CLUSTER", 1);
  if (plan.nwm == 0 && plan.nwk <= 4 && !dense && can_split && plan.n_chunks >= 2 && plan.n_chunks <= 8 &&
      cl_mode != 0) {
    const bool one_wave = plan.n_units * plan.n_chunks <= sm_count_cached() * n8_resident_per_sm(a, plan.variant);
    if (cl_mode == 2 || one_wave) plan.cluster = 1;
  }
  if (dense && !ext && ct > kMaxChunkTiles) {
    // The per-CTA page table holds kMaxChunkTiles entries; a dense sequence longer
    // than that is still one page, so only its first entry is read -- but keep the
    // table bound honest by splitting into several single-page chunks is not allowed
    // without workspace.  Fall back to the generic kernel.
    return plan;
  }
  plan.ws_bytes = 0;
  if (plan.n_chunks > 1 && !plan.cluster) {
    plan.ws_bytes = kCounterBytes + align256(plan.n_units * plan.n_chunks * plan.rows_real * sizeof(float2)) +
                    (size_t)plan.n_units * plan.n_chunks * plan.rows_real * a.D * sizeof(float);
  }
  plan.eligible = true;
  return plan;
}

size_t mma_ws_ml() { return kCounterBytes; }
size_t mma_ws_o(const MmaPlan& plan) {
  return kCounterBytes + align256(plan.n_units * plan.n_chunks * plan.rows_real * sizeof(float2));
}

int launch_paged_mma(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  if (paged_is_ext(a)) return launch_paged_mma_window(a, plan, ws, s);
  if (a.kv_dtype == NVM_F16) {
    return a.D == 64 ? launch_d<__half, __half, 64>(a, plan, ws, s) : launch_d<__half, __half, 128>(a, plan, ws, s);
  }
  if (a.kv_dtype == NVM_BF16) {
    return a.D == 64 ? launch_d<__nv_bfloat16, __nv_bfloat16, 64>(a, plan, ws, s)
                     : launch_d<__nv_bfloat16, __nv_bfloat16, 128>(a, plan, ws, s);
  }
  if (a.scale_dtype == NVM_F16) return launch_d<int8_t, __half, 128>(a, plan, ws, s);
  return launch_d<int8_t, __nv_bfloat16, 128>(a, plan, ws, s);
}

}  // namespace nvm
