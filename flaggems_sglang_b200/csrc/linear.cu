// Dense products of e4m3 operands with a scale per 128 channels of every token and per 128 x 128 block of the weights:
//     y[t, n] = sum_kb a[t, kb] * b[n / 128, kb] * (sum_{k in kb} xq[t, k] * wq[n, k])
// what a layer computes beside its routed experts (shared expert, attention projections).
//
// The tensor cores cannot apply a scale inside their accumulator that changes with K, so every K block of 128 is multiplied into
// a fresh TMEM partial (4 MMAs of K = 32) which the fold warps add, times a[t, kb] * b[n / 128, kb], to sums in registers.
//
//   tile    : 128 weight rows x up to 16, 32 or 64 tokens, the weights on the MMA's M side, so that one token costs a 16-column tile; or
//             x up to 128 tokens with the tokens on M, where a fold thread owns a token and needs one factor per K block instead of one per
//             column (128 tokens, 7168 x 4096, unsplit: 27 -> 18 us)
//   gate/up : a tile is 128 channels, 64 gate rows and the same channels' up rows in each of two CTAs of the cluster
//   split   : S CTAs (gate/up: S pairs) of a cluster share a tile, each with a contiguous part of its K blocks, so that few tiles still
//             fill the chip.  Their sums meet through distributed shared memory, added in the order of the CTAs: the result does not
//             depend on timing, and there is no scratch in global memory and no counter.  Up to 64 tokens every CTA sends its sums to the
//             ones that store them (st.async, one mbarrier there; against two cluster barriers and reading the others' memory one token
//             of 7168 x 2048 4.7 -> 4.2 us, 16 tokens of 2048 x 7168 5.1 -> 4.2); tiles of 128 tokens keep theirs, which
//             the others read (sent, 128 tokens of 2048 x 7168 took 8.4 us against 7.5)
//   warps   : fold warps (TMEM lane quarter = warp % 4; 16 or 32 sums per thread), then TMA, MMA, and two that multiply token and weight
//             scales into a ring of factors
//   batches : up to 32 tokens the partials of two or four K blocks are handed to the fold together.  What a K block costs there is not
//             its FMAs but the chain wait - TMEM read - wait - hand back: 400 SM cycles each alone, 180 in batches of four
//   epilogue: a warp per token: a row of 128 channels is one coalesced store, and for
//             gate/up it is one quantisation group, whose largest magnitude is a warp reduction
//   bf16    : tokens are quantised by this kernel's idle warps while the weights are on their way, where the rows of a CTA are few: every
//             CTA of a row of tiles quantises them again, some 25 instructions per channel, against 2.2 us for a launch that does it once
//             (one token of 7168 x 2048 6.6 -> 5.5 us, 8 tokens of 2048 x 7168 6.4 -> 5.7; 16 of these 6.5 -> 7.3, so they are not)
// Up to 32 tokens two CTAs share an SM: twice as many clusters of 8 fit.  (A register limit of 80 per thread, which two CTAs of 384 threads
// or gate and up rows in one CTA bring, makes the fold take twice as long: 64 tokens 38 us for 56 K blocks against 17.7 with one CTA.)
// Every mbarrier wait is bounded; the cluster barriers are reached by every thread on every path.
// What bounds it: up to 64 tokens HBM beside the launch, the first loads and the join (one token, 7168 x 4096: 6.2 us, 4.7 TB/s; gate/up of
// 7168 x 2 x 2048 6.6 us); with 128 tokens shared memory, 32 KB in and 32 KB of operands per K block (0.27 us).
#include "linear.cuh"
#include "pair.cuh"
#include "rows.cuh"

#include <algorithm>
#include <mutex>

namespace fmoe {

// This translation unit's status word; read by status_word_linear().
__device__ int g_device_status_linear = 0;

namespace {

constexpr int KBYTES = 128;
constexpr int W_BYTES = 128 * KBYTES;
constexpr int kMaxStages = 12;
constexpr int kGroup = 8;  // K blocks per factor slot
constexpr int kSlots = 4;
constexpr int kMaxSplit = 8;
constexpr int BAR_BYTES = 512;

// COLS: most tokens of a tile; BATCH: K blocks whose partials are handed to the fold together; ACC: sums per fold thread; CTAS: CTAs per SM;
// TOKENS_M: the tokens on M
template <int COLS_, int BATCH_, int ACC_, int CTAS_, bool TOKENS_M_>
struct Geo {
  static constexpr int COLS = COLS_, BATCH = BATCH_, ACC = ACC_, CTAS = CTAS_;
  static constexpr bool TOKENS_M = TOKENS_M_;
  static constexpr int FOLD_WARPS = 4 * (TOKENS_M ? 128 : COLS) / ACC;
  static constexpr int THREADS = (FOLD_WARPS + 4) * 32;
  static constexpr int BUF_COLS = TOKENS_M ? 128 : BATCH * COLS;  // TMEM columns of a batch's partials
  static constexpr int BUFS = 512 / CTAS / BUF_COLS < 4 ? 512 / CTAS / BUF_COLS : 4;
  static constexpr int TMEM_COLS = BUFS * BUF_COLS;
  // what a CTA takes, whatever its ring needs: so that neither a third CTA nor another TMEM kernel fits beside these, whose TMEM
  // allocation would wait for this one's end while a cluster of its own waits for it
  static constexpr int SMEM_BYTES = CTAS == 1 ? 227 * 1024 : 113 * 1024;
  // Sums: up to 64 tokens every CTA sends its own to the CTAs that store them, which have room for them beside the ring: 128 floats per
  // token and sender.  TOKENS_M: they stay here, in place of the ring, four floats of shift from token to token for the 16-byte stores of
  // the fold, and are read by the CTAs that store them.
  static constexpr bool SENDS = !TOKENS_M;
  static constexpr int SUM_PITCH = 128 + (TOKENS_M ? 4 : 0);
  static constexpr int LAND_BYTES = SENDS ? (COLS + kMaxSplit) * 512 : 0;
  static constexpr int SUM_BYTES = SENDS ? 0 : COLS * SUM_PITCH * 4;
  // factors of one K block: [gated: gate rows | up rows][token]
  static constexpr int kb_floats(bool gated) { return (gated ? 2 : 1) * COLS; }
  static constexpr int fixed_bytes(bool gated) { return BAR_BYTES + LAND_BYTES + kSlots * kGroup * kb_floats(gated) * 4; }
  static_assert(SUM_BYTES <= SMEM_BYTES - fixed_bytes(true) && TMEM_COLS * CTAS <= 512 && kGroup % BATCH == 0, "shared memory, TMEM");
};

struct KernelParams {
  const float* x_scale;
  const __nv_bfloat16* x_bf16;  // QUANT
  const float* w_scale;
  const float* bias;
  const __nv_bfloat16* addend;
  void* out;
  float* out_scale;
  int64_t T, n;
  int kblocks;
  int token_tiles, token_tile;  // token_tile: a multiple of 16
  int stages, stage_bytes;
  int token_bytes;  // QUANT: a K block of the tile's tokens
  int split;      // CTAs that share a tile's K blocks (gated: pairs of CTAs, each with half of the tile's channels)
  int activation;
  int early;      // the weights are complete when the kernel starts
};

__device__ __forceinline__ void report(int code) { atomicCAS(&g_device_status_linear, 0, code); }

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity));
}

// QUANT: the tokens are bf16 and quantised here, into an area behind the ring that holds all K blocks of this CTA
template <typename G, bool GATED, bool QUANT>
__global__ void __launch_bounds__(G::THREADS, G::CTAS)
fp8_linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const KernelParams p) {
  constexpr int COLS = G::COLS, BATCH = G::BATCH, KB_FLOATS = G::kb_floats(GATED), SLOT_FLOATS = kGroup * KB_FLOATS;
  extern __shared__ __align__(1024) uint8_t smem[];
  // barriers and factors behind the ring; the ring starts at 0 (1024-byte aligned stages: weights, then tokens)
  uint8_t* fixed = smem + G::SMEM_BYTES - G::fixed_bytes(GATED);
  uint64_t* bars = reinterpret_cast<uint64_t*>(fixed);
  uint64_t* full_bar = bars;                    // [stages] TMA -> MMA
  uint64_t* empty_bar = bars + kMaxStages;      // [stages] MMA -> TMA
  uint64_t* part_full = bars + 2 * kMaxStages;  // [BUFS] MMA -> fold
  uint64_t* part_empty = part_full + 4;         // [BUFS] fold -> MMA
  uint64_t* sc_full = part_empty + 4;           // [kSlots] factor warps -> fold
  uint64_t* sc_empty = sc_full + kSlots;        // [kSlots] fold -> factor warps
  uint64_t* land_bar = sc_empty + kSlots;       // [1] sums of all CTAs -> epilogue
  uint64_t* quant_bar = land_bar + 1;           // [1] quantisers -> MMA, fold
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(quant_bar + 1);
  uint8_t* land = fixed + BAR_BYTES;
  float* factors = reinterpret_cast<float*>(land + G::LAND_BYTES);

  const int warp = ptx::uniform_warp_id(), lane = threadIdx.x & 31;
  const int S = p.split, ctas = GATED ? 2 * S : S;  // of a cluster
  const int rank = ctas > 1 ? (int)ptx::cluster_ctarank() : 0;
  const int slice = GATED ? rank >> 1 : rank, side = GATED ? rank & 1 : 0;  // part of K, half of the channels
  const int tile = (int)blockIdx.x / ctas;
  const int row_tile = tile / p.token_tiles;
  const int tok0 = tile % p.token_tiles * p.token_tile;
  const int kb0 = (int)((int64_t)p.kblocks * slice / S), kb1 = (int)((int64_t)p.kblocks * (slice + 1) / S);
  const int up_tile = row_tile + (int)(p.n / 128);  // gated: the tile of up rows

  const int tokens = (int)min((int64_t)p.token_tile, p.T - tok0);
  const int mine = (tokens - rank + ctas - 1) / ctas;  // this CTA stores the tokens rank, rank + ctas, ..
  if (threadIdx.x < 32) {
    if (lane < p.stages) {
      ptx::mbar_init(&full_bar[lane], 1);
      ptx::mbar_init(&empty_bar[lane], 1);
    }
    if (lane < G::BUFS) {
      ptx::mbar_init(&part_full[lane], 1);
      ptx::mbar_init(&part_empty[lane], G::FOLD_WARPS);
    }
    if (lane < kSlots) {
      ptx::mbar_init(&sc_full[lane], 1);
      ptx::mbar_init(&sc_empty[lane], G::FOLD_WARPS);
    }
    if (lane == 0) {
      ptx::mbar_init(land_bar, 1);
      if (QUANT) ptx::mbar_init(quant_bar, G::FOLD_WARPS + 2);
      if (G::SENDS && ctas > 1) ptx::mbar_arrive_expect_tx(land_bar, mine * ctas * 512);
    }
    ptx::fence_barrier_init();
  }
  if (warp == G::FOLD_WARPS && lane == 0) {
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_w);
  }
  if (warp == G::FOLD_WARPS + 1) {
    ptx::tmem_alloc(tmem_slot, G::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  if (G::SENDS && ctas > 1) ptx::cluster_arrive();  // and waited for before the first sums are sent
  const uint32_t tmem_base = *tmem_slot;

  if (!GATED && p.addend && warp == G::FOLD_WARPS + 3) {  // on its way to L2 while the tile is multiplied: the tokens that this CTA will store
    pdl_wait();
    const int64_t ch = (int64_t)row_tile * 128;
    const int lines = (int)(min((int64_t)128, p.n - ch) * 2 + 127) / 128;
    for (int t = rank + ctas * lane; t < p.token_tile && tok0 + t < p.T; t += ctas * 32)
      for (int l = 0; l < lines; ++l) prefetch_l2(reinterpret_cast<const uint8_t*>(p.addend + (tok0 + t) * p.n + ch) + 128 * l);
  }
  if constexpr (QUANT) {
    static_assert(!G::TOKENS_M, "built for up to 64 tokens");
    // ---------------- tokens: eight lanes own a group of 128 channels, all warps but those of TMA and MMA ----------------
    if (warp < G::FOLD_WARPS || warp >= G::FOLD_WARPS + 2) {
      pdl_entry_late();
      constexpr int kIlp = 4, TEAMS = (G::FOLD_WARPS + 2) * 4;
      const int sub = lane & 7, team = (warp < G::FOLD_WARPS ? warp : warp - 2) * 4 + (lane >> 3);
      const int items = tokens * (kb1 - kb0);  // K block by K block
      uint8_t* area = smem + p.stages * p.stage_bytes;
      for (int first = team; __any_sync(0xffffffffu, first < items); first += TEAMS * kIlp) {
        uint4 raw[kIlp][2];
        float w[kIlp];  // of the weight block, in the lane that will write the factor
        int at[kIlp], kbs[kIlp];
#pragma unroll
        for (int u = 0; u < kIlp; ++u) {
          const int i = first + u * TEAMS;
          kbs[u] = i / tokens;
          at[u] = i - kbs[u] * tokens;
          raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
          w[u] = 0.f;
          if (i < items) {
            const uint4* src = reinterpret_cast<const uint4*>(p.x_bf16 + ((tok0 + at[u]) * (int64_t)p.kblocks + kb0 + kbs[u]) * 128) + sub * 2;
            raw[u][0] = __ldg(src);
            raw[u][1] = __ldg(src + 1);
            if (sub < (GATED ? 2 : 1)) w[u] = __ldg(p.w_scale + (int64_t)(sub ? up_tile : row_tile) * p.kblocks + kb0 + kbs[u]);
          }
        }
        uint4 packed[kIlp];
        float s[kIlp];
        quant_groups(raw, packed, s);
#pragma unroll
        for (int u = 0; u < kIlp; ++u) {
          if (first + u * TEAMS < items) {  // the swizzle of a 128-byte row: its 16-byte pieces exchanged by the row's number
            *reinterpret_cast<uint4*>(area + kbs[u] * p.token_bytes + at[u] * KBYTES + ((sub ^ (at[u] & 7)) << 4)) = packed[u];
            if (sub < (GATED ? 2 : 1)) factors[kbs[u] * KB_FLOATS + sub * COLS + at[u]] = s[u] * w[u];
          }
        }
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(quant_bar);
    }
  }

  if (warp == G::FOLD_WARPS) {
    // ---------------- TMA producer ----------------
    if (ptx::elect_one()) {
      const uint32_t ring = ptx::smem_u32(smem);
      const uint32_t bytes = QUANT ? W_BYTES : W_BYTES + p.token_tile * KBYTES;
      auto load_weights = [&](int kb, int s) {
        const uint32_t dst = ring + s * p.stage_bytes, bar = ptx::smem_u32(&full_bar[s]);
        ptx::mbar_arrive_expect_tx(&full_bar[s], bytes);
        if constexpr (GATED) {  // 64 gate rows, then the same channels' up rows
          ptx::tma_load_2d(dst, &map_w, kb * KBYTES, row_tile * 128 + side * 64, bar);
          ptx::tma_load_2d(dst + W_BYTES / 2, &map_w, kb * KBYTES, up_tile * 128 + side * 64, bar);
        } else {
          ptx::tma_load_2d(dst, &map_w, kb * KBYTES, row_tile * 128, bar);
        }
      };
      auto load_tokens = [&](int kb, int s) {
        if constexpr (!QUANT) ptx::tma_load_2d(ring + s * p.stage_bytes + W_BYTES, &map_x, kb * KBYTES, tok0, ptx::smem_u32(&full_bar[s]));
      };
      int kb = kb0, stage = 0;
      uint32_t phase = 0;
      if (p.early) {  // weights that nothing before this kernel writes are on their way before the tokens are there
        const int ahead = min(p.stages, kb1 - kb0);
        for (int s = 0; s < ahead; ++s) load_weights(kb0 + s, s);
        pdl_wait();
        for (int s = 0; s < ahead; ++s) load_tokens(kb0 + s, s);
        kb += ahead;
        if (ahead == p.stages) phase = 1;
        else stage = ahead;
      } else {
        pdl_wait();
      }
      pdl_trigger();
      for (; kb < kb1; ++kb) {
        if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1)) {
          report(0x1100 | stage);
          break;
        }
        load_weights(kb, stage);
        load_tokens(kb, stage);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // nothing is in flight when this CTA ends or its sums take the ring's place
      for (int left = min(p.stages, kb - kb0); left > 0; --left) {
        if (--stage < 0) {
          stage = p.stages - 1;
          phase ^= 1;
        }
        if (!ptx::mbar_wait(&full_bar[stage], phase)) report(0x1140 | stage);
      }
    }
    __syncwarp();
  } else if (warp == G::FOLD_WARPS + 1) {
    // ---------------- MMA issuer: one fresh partial per K block ----------------
    if (ptx::elect_one()) {
      pdl_wait();
      pdl_trigger();
      const uint32_t ring = ptx::smem_u32(smem);
      const uint64_t dw0 = ptx::smem_desc_sw128(ring), dx0 = ptx::smem_desc_sw128(ring + (QUANT ? p.stages * p.stage_bytes : W_BYTES));
      const uint32_t idesc = ptx::make_idesc(/*e4m3*/ 0, 128, G::TOKENS_M ? 128 : (uint32_t)p.token_tile);
      int stage = 0;
      uint32_t phase = 0;
      int steps = kb1 - kb0;
      if (QUANT && !ptx::mbar_wait(quant_bar, 0)) {
        report(0x1280);
        steps = 0;
      }
      for (int step = 0; step < steps; ++step) {
        const int batch = step / BATCH, buf = batch % G::BUFS;
        if (!ptx::mbar_wait(&full_bar[stage], phase)) {
          report(0x1200 | stage);
          break;
        }
        if (step % BATCH == 0 && !ptx::mbar_wait(&part_empty[buf], ((batch / G::BUFS) & 1) ^ 1)) {
          report(0x1240 | buf);
          break;
        }
        ptx::tc_fence_after_sync();
        const uint64_t off = (uint64_t)(stage * (p.stage_bytes >> 4)), dw = dw0 + off;
        const uint64_t dx = dx0 + (QUANT ? (uint64_t)(step * (p.token_bytes >> 4)) : off);
        const uint32_t to = tmem_base + buf * G::BUF_COLS + (G::TOKENS_M ? 0 : step % BATCH * COLS);
#pragma unroll
        for (int kk = 0; kk < KBYTES / 32; ++kk)
          ptx::mma_f8f6f4_ss(to, (G::TOKENS_M ? dx : dw) + 2 * kk, (G::TOKENS_M ? dw : dx) + 2 * kk, idesc, kk != 0);
        if (step % BATCH == BATCH - 1 || step == steps - 1) ptx::mma_commit(&part_full[buf]);
        ptx::mma_commit(&empty_bar[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp >= G::FOLD_WARPS + 2) {
    // ---------------- factors: two warps take alternate groups of eight K blocks ----------------
    pdl_entry_late();
    const int me = warp - (G::FOLD_WARPS + 2);
    for (int g = me; !QUANT && g * kGroup < kb1 - kb0; g += 2) {
      const int first = kb0 + g * kGroup, count = min(kGroup, kb1 - first), slot = g % kSlots;
      constexpr int PER_LANE = (COLS + 31) / 32;
      constexpr int ROW_BLOCKS = GATED ? 2 : 1;
      float a[PER_LANE][kGroup], b[ROW_BLOCKS][kGroup];
#pragma unroll
      for (int h = 0; h < ROW_BLOCKS; ++h) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) b[h][i] = i < count ? __ldg(p.w_scale + (int64_t)(h ? up_tile : row_tile) * p.kblocks + first + i) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        const int64_t t = tok0 + lane + 32 * j;
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          a[j][i] = (lane + 32 * j < p.token_tile && t < p.T && i < count) ? __ldg(p.x_scale + t * p.kblocks + first + i) : 0.f;
      }
      if (!warp_wait(&sc_empty[slot], ((g / kSlots) & 1) ^ 1)) {
        report(0x1300 | slot);
        break;
      }
      float* dst = factors + slot * SLOT_FLOATS + lane;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
#pragma unroll
        for (int h = 0; h < ROW_BLOCKS; ++h) {
#pragma unroll
          for (int j = 0; j < PER_LANE; ++j)
            if (COLS % 32 == 0 || lane < COLS) dst[i * KB_FLOATS + h * COLS + 32 * j] = a[j][i] * b[h][i];
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sc_full[slot]);
    }
  } else if constexpr (G::TOKENS_M) {
    // ---------------- fold: a thread has a token, so one factor per half ----------------
    pdl_entry_late();
    constexpr int ACC = G::ACC;
    static_assert(!G::TOKENS_M || ACC == 32, "one read per K block");
    const int piece = warp >> 2, tok = (warp & 3) * 32 + lane;
    const uint32_t from = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + piece * ACC;
    const float* mine = factors + (GATED ? piece >> 1 : 0) * COLS + tok;
    float acc[ACC];
#pragma unroll
    for (int i = 0; i < ACC; ++i) acc[i] = 0.f;
    const int steps = kb1 - kb0;
    for (int step = 0; step < steps; ++step) {
      const int buf = step % G::BUFS, g = step / kGroup, slot = g % kSlots;
      if (step % kGroup == 0 && !warp_wait(&sc_full[slot], (g / kSlots) & 1)) {
        report(0x1480 | slot);
        break;
      }
      const float f = mine[slot * SLOT_FLOATS + step % kGroup * KB_FLOATS];
      if (!warp_wait(&part_full[buf], (step / G::BUFS) & 1)) {
        report(0x14c0 | buf);
        break;
      }
      ptx::tc_fence_after_sync();
      uint32_t v[32];
      ptx::tmem_ld_32x32b_x32(from + buf * G::BUF_COLS, v);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      ptx::mbar_arrive_if(lane == 0, &part_empty[buf]);
#pragma unroll
      for (int i = 0; i < ACC; ++i) acc[i] = fmaf(__uint_as_float(v[i]), f, acc[i]);
      if (step % kGroup == kGroup - 1 || step == steps - 1) ptx::mbar_arrive_if(lane == 0, &sc_empty[slot]);
    }
    // sums to shared memory, as below
    float* sums = reinterpret_cast<float*>(smem) + tok * G::SUM_PITCH + piece * ACC;
    if (tok < p.token_tile) {
#pragma unroll
      for (int i = 0; i < ACC; i += 4) *reinterpret_cast<float4*>(sums + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    }
  } else {
    // ---------------- fold ----------------
    pdl_entry_late();
    constexpr int ACC = G::ACC;
    const int col0 = (warp >> 2) * ACC;
    const int cols = min(ACC, p.token_tile - col0);  // a multiple of 16, or nothing
    const uint32_t from = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + col0;
    const float* mine = factors + (GATED ? (warp & 3) >> 1 : 0) * COLS + col0;  // gated: lanes 0-63 hold gate rows
    float acc[ACC];
#pragma unroll
    for (int i = 0; i < ACC; ++i) acc[i] = 0.f;
    int steps = kb1 - kb0;
    if (QUANT && !warp_wait(quant_bar, 0)) {  // all factors are there
      report(0x15c0);
      steps = 0;
    }
    for (int step = 0; step < steps; step += BATCH) {
      const int batch = step / BATCH, buf = batch % G::BUFS, g = step / kGroup, slot = g % kSlots, blocks = min(BATCH, steps - step);
      if (!QUANT && step % kGroup == 0 && !warp_wait(&sc_full[slot], (g / kSlots) & 1)) {
        report(0x1400 | slot);
        break;
      }
      if (!warp_wait(&part_full[buf], (batch / G::BUFS) & 1)) {
        report(0x1440 | buf);
        break;
      }
      ptx::tc_fence_after_sync();
      const float* f = mine + slot * SLOT_FLOATS + step % kGroup * KB_FLOATS;
      // The batch's columns, ACC of each K block in turn: all are read before the first is waited for, and the partials are handed back
      // before the FMAs, so that the MMAs of later K blocks run beside them.
      constexpr int ALL = BATCH * ACC;
      auto there = [&](int q) { return q / ACC < blocks && q % ACC < cols; };
      uint32_t v[ALL];
#pragma unroll
      for (int q = 0; q < ALL; q += 16)
        if (there(q)) ptx::tmem_ld_32x32b_x16(from + buf * G::BUF_COLS + q / ACC * COLS + q % ACC, *reinterpret_cast<uint32_t(*)[16]>(v + q));
      ptx::tmem_ld_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      ptx::mbar_arrive_if(lane == 0, &part_empty[buf]);
#pragma unroll
      for (int q = 0; q < ALL; q += 4) {
        if (there(q & ~15)) {
          const float4 f4 = *reinterpret_cast<const float4*>(f + q / ACC * KB_FLOATS + q % ACC);
          float* d = acc + q % ACC;
          d[0] = fmaf(__uint_as_float(v[q]), f4.x, d[0]);
          d[1] = fmaf(__uint_as_float(v[q + 1]), f4.y, d[1]);
          d[2] = fmaf(__uint_as_float(v[q + 2]), f4.z, d[2]);
          d[3] = fmaf(__uint_as_float(v[q + 3]), f4.w, d[3]);
        }
      }
      if (step % kGroup == kGroup - BATCH || step + BATCH >= steps) {
        __syncwarp();
        ptx::mbar_arrive_if(lane == 0, &sc_empty[slot]);
      }
    }
    // A warp has 32 consecutive rows of its tokens: through shared memory (in place of the ring: the last partial is complete, so every MMA
    // has read its operands) into 16-byte pieces, and these to the CTA that stores the token, whose j-th token's sums from sender r are at
    // land + (j * ctas + r) * 512.  (4 bytes at a time: 16 tokens 8.5 us where this takes 7.1.)
    float* sums = reinterpret_cast<float*>(ctas > 1 ? smem : land) + (warp & 3) * 32;
#pragma unroll
    for (int i = 0; i < ACC; ++i)
      if (i < cols) sums[(col0 + i) * 128 + lane] = acc[i];
    if (ctas > 1) {
      __syncwarp();
      ptx::cluster_wait();
      const uint32_t to = ptx::smem_u32(land) + rank * 512 + ((warp & 3) * 32 + (lane & 7) * 4) * 4, bar = ptx::smem_u32(land_bar);
      for (int t = col0 + (lane >> 3); t < min(col0 + cols, tokens); t += 4) {
        const int j = t / ctas, owner = t - j * ctas;
        ptx::st_async_f4(ptx::mapa(to + j * ctas * 512, owner), *reinterpret_cast<const float4*>(sums + t * 128 + (lane & 7) * 4),
                         ptx::mapa(bar, owner));
      }
      __syncwarp();
    }
  }

  ptx::tc_fence_before_sync();
  if (!G::SENDS && ctas > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp == G::FOLD_WARPS + 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, G::TMEM_COLS);
  }

  // ---------------- epilogue: a warp per token, the tile's tokens dealt to the CTAs of the cluster ----------------
  auto store = [&](int t, auto& v) {
    const int64_t row = tok0 + t;
    if constexpr (GATED) {
      store_gated(v, p.activation, reinterpret_cast<uint8_t*>(p.out) + row * p.n + row_tile * 128, p.out_scale + row * (p.n / 128) + row_tile);
    } else {
      const int64_t ch = (int64_t)row_tile * 128 + lane * 4;
      if (ch < p.n) store_plain(v[0], p.bias, p.addend, reinterpret_cast<__nv_bfloat16*>(p.out), row * p.n, ch);
    }
  };
  constexpr int ROW_BLOCKS = GATED ? 2 : 1;
  if constexpr (G::SENDS) {
    if (ctas > 1) {
      if (mine > 0 && !warp_wait(land_bar, 0)) {
        report(0x1500);
        warp_wait(land_bar, 0);  // nobody writes here after this CTA has left
      }
      if (warp >= G::FOLD_WARPS) ptx::cluster_wait();  // the warps that sent nothing complete the barrier of the beginning
    }
    // gated: the sums of 64 channels' gate and up rows come from every second sender; lanes 0-15 take the first half's, 16-31 the second's
    const float* at = reinterpret_cast<const float*>(land) + (GATED ? (lane >> 4) * 128 + (lane & 15) * 4 : lane * 4);
    for (int j = warp; j < mine; j += G::THREADS / 32) {
      float v[ROW_BLOCKS][4];
#pragma unroll
      for (int h = 0; h < ROW_BLOCKS; ++h) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[h][q] = 0.f;
      }
      for (int s = 0; s < S; ++s) {  // in the order of the senders
#pragma unroll
        for (int h = 0; h < ROW_BLOCKS; ++h) {
          const float4 part = *reinterpret_cast<const float4*>(at + (j * ctas + s * ROW_BLOCKS) * 128 + 64 * h);
          v[h][0] += part.x;
          v[h][1] += part.y;
          v[h][2] += part.z;
          v[h][3] += part.w;
        }
      }
      store(rank + j * ctas, v);
    }
  } else {
    const uint32_t sums = ptx::smem_u32(smem);
    const int first = rank + ctas * warp, stride = ctas * (G::THREADS / 32);
    if constexpr (GATED)  // as above
      join_tokens<2, kMaxSplit / 2>(first, stride, tokens, S, lane >> 4, 2, true, sums + (lane & 15) * 16, G::SUM_PITCH * 4, 256, store);
    else join_tokens<1, kMaxSplit>(first, stride, tokens, S, 0, 1, S > 1, sums + lane * 16, G::SUM_PITCH * 4, 0, store);
    if (ctas > 1) ptx::cluster_sync_relaxed();  // nobody leaves while its sums are read
  }
}

using Few = Geo<16, 4, 16, 2, false>;
using Some = Geo<32, 2, 32, 2, false>;
using Half = Geo<64, 1, 32, 1, false>;
using Many = Geo<128, 1, 32, 1, true>;

// The query below counts one CTA per SM for every kernel that allocates TMEM, whatever it takes, so it is asked about this one, with the
// others' shared memory and threads.
__global__ void __launch_bounds__(Many::THREADS) stand_in_kernel() {}

// Clusters of 1 to 8 CTAs that the device holds at a time, by the CTAs per SM.  GPCs have different numbers of SMs, so that clusters of
// 7 or 8 leave a fifth of them idle where a CTA takes a whole SM.
struct Residents {
  int n[2][kMaxSplit + 1];
};

const Residents& residents() {
  static std::mutex mu;
  static Residents known[kMaxDevices];
  static bool done[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) dev = 0;
  std::lock_guard<std::mutex> lock(mu);
  Residents& r = known[dev];
  if (!done[dev]) {
    auto ask = [](int threads, int smem, int split) {
      cudaFuncSetAttribute(stand_in_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(split);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = split;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, stand_in_kernel, &cfg) == cudaSuccess && n > 0) return n;
      cudaGetLastError();
      return 0;
    };
    for (int s = 1; s <= kMaxSplit; ++s) {
      r.n[0][s] = ask(Many::THREADS, Many::SMEM_BYTES, s);
      r.n[1][s] = ask(Few::THREADS, Few::SMEM_BYTES, s);
      for (int c = 0; c < 2; ++c)
        if (r.n[c][s] == 0) r.n[c][s] = std::max(1, 148 * (c + 1) / s);
    }
    done[dev] = true;
  }
  return r;
}

// The kernel and the number of CTAs (pair kernel: pairs) that share a tile's K blocks, by what the launch should take.  The models were
// fitted to launches of K = 2048, 4096 and 7168, N = 512 to 7168 (gate/up: I = 768 to 3584) and 1 to 1024 tokens with every split; us:
//   one CTA    rounds of clusters, each its K blocks at the slowest of the fold (0.19 to 0.28 by width), HBM's share of the weights and
//              what an SM and the chip take in from L2, an epilogue, and the join of the sums; more than half the chip's room is dearer,
//              as the next launch then cannot begin beside this one
//   bf16 rows  2.2 for the quantiser's launch, or 0.9 (1.7 where CTAs share SMs) and 0.3 for every group of 128 channels that eight lanes
//              quantise in the kernel; behind another launch of the same call clusters of 8 take 1.0 longer
//   CTA pairs  rounds of 0.38 per K block and the epilogue; shared tiles 0.44 and a longer one, as all sums cross shared memory
// The choice takes 1.01 times the best of all kernels and splits on average of 112 products, 1.10 times at worst, 1.00 times of 64 gate/up products,
// 1.01 (1.05) times of 36 products of bf16 rows; 1 to 2048 tokens.
struct Choice {
  bool pair;
  int split;
  bool quant;  // the one-CTA kernel quantises bf16 tokens itself
};

thread_local Choice t_debug_choice{false, 0, false};  // fmoe_debug_linear_kernel

int token_tile_of(int64_t T, int cols) {
  const int64_t tiles = ceil_div<int64_t>(T, cols);
  return (int)(ceil_div<int64_t>(ceil_div<int64_t>(T, tiles), 16) * 16);
}

// Stages of weights beside the quantised tokens of `slice` K blocks; 0: too few to keep the loads going, or no room for the factors
template <typename G>
int quant_stages(bool gated, int token_tile, int slice) {
  const int token_bytes = token_tile * KBYTES;
  if (slice > kSlots * kGroup) return 0;
  const int stages = std::min(std::min(kMaxStages, slice), (G::SMEM_BYTES - G::fixed_bytes(gated) - slice * token_bytes) / W_BYTES);
  return stages < std::min(slice, 4) ? 0 : stages;
}
bool can_quant(int64_t T, bool gated, int slice) {
  if (T <= 16) return quant_stages<Few>(gated, 16, slice) > 0;
  if (T <= 32) return quant_stages<Some>(gated, 32, slice) > 0;
  return T <= 64 && quant_stages<Half>(gated, token_tile_of(T, 64), slice) > 0;
}

Choice choose(const LinearParams& g, bool gated) {
  const Residents& r = residents();
  const int kblocks = (int)(g.k / 128);
  const int cols = g.T <= 16 ? 16 : (g.T <= 32 ? 32 : (g.T <= 64 ? 64 : 128));
  const int ctas = cols <= 32 ? 2 : 1, sides = gated ? 2 : 1;
  const int64_t token_tiles = ceil_div<int64_t>(g.T, cols), tiles = ceil_div<int64_t>(g.n, 128) * token_tiles;
  const double tokens = (double)(ceil_div<int64_t>(ceil_div<int64_t>(g.T, token_tiles), 16) * 16);
  const double fold = cols == 128 ? 0.28 : 0.17 + 0.001 * cols;
  const double bytes = W_BYTES + tokens * KBYTES;
  Choice best{false, 1, false};
  double best_us = 1e30;
  auto offer = [&](bool pair, int split, double us, bool quant = false) {
    if (us < best_us) {
      best_us = us;
      best = {pair, split, quant};
    }
  };
  const double before = g.x_bf16 ? 2.2 : 0.0;  // a quantiser's launch
  for (int s = 1; s * sides <= kMaxSplit && s <= kblocks; ++s) {
    if (s == 7) continue;  // fits the GPCs badly: never more than 2 % better than another
    const int64_t at_once = r.n[ctas - 1][s * sides], rounds = ceil_div<int64_t>(tiles, at_once);
    const double active = (double)std::min<int64_t>(tiles, at_once) * s * sides, per_sm = std::max(1.0, active / 148);
    const double hbm = active * W_BYTES / (gated ? 12.0e6 : 8.0e6), l2 = std::max(bytes * per_sm / 1.2e5, active * bytes / 1.5e7);
    const double per_block = std::max(std::max(hbm, l2), fold * per_sm);
    const double join = s == 1 ? 0.0 : 0.2 + 0.05 * s + (gated ? 0.004 : 0.008) * tokens;
    const double us = (active > 74 * ctas ? 2.4 : 2.0) + rounds * (0.7 + 0.01 * tokens + (gated ? 0.9 : 0.0) + (rounds > 1 ? 1.2 : 0.0) + ceil_div(kblocks, s) * per_block + join);
    const bool wide = s == 8 && !gated;  // clusters that come in late while another launch leaves
    offer(false, s, us + before + (wide && (g.x_bf16 || g.behind_late_trigger) ? 1.0 : 0.0));
    if (g.x_bf16 && can_quant(g.T, gated, ceil_div(kblocks, s))) offer(false, s, us + rounds * ((active > 148 ? 1.7 : 0.9) + 0.3 * g.T * ceil_div(kblocks, s) / (cols == 64 ? 40 : 24)), true);
  }
  if (g.T > 64) {
    const int64_t pair_tiles = ceil_div<int64_t>(g.T, 256) * ceil_div<int64_t>(g.n, gated ? 128 : 256);
    offer(true, 1, before + 3.0 + ceil_div<int64_t>(pair_tiles, r.n[0][2]) * (0.38 * kblocks + 3.0));
    for (int s = 2; s <= kMaxPairSplit && s <= kblocks; ++s)
      offer(true, s, before + 2.8 + ceil_div<int64_t>(pair_tiles, r.n[0][2 * s]) * (0.44 * ceil_div(kblocks, s) + 5.7));
  }
  return best;
}

template <typename G, bool GATED, bool QUANT>
int launch(const LinearParams& g, int split, cudaStream_t st) {
  auto kernel = fp8_linear_kernel<G, GATED, QUANT>;
  static PerDeviceOnce once_attr;
  const cudaError_t attr_err = per_device_once(once_attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM_BYTES);
  });
  if (attr_err != cudaSuccess) return fail(FMOE_ERR_CUDA, "set-up of the e4m3 linear kernel failed: %s", cudaGetErrorString(attr_err));
  KernelParams p;
  p.token_tiles = (int)ceil_div<int64_t>(g.T, G::COLS);
  p.token_tile = token_tile_of(g.T, G::COLS);
  p.token_bytes = (G::TOKENS_M ? G::COLS : p.token_tile) * KBYTES;  // TOKENS_M: lanes without tokens multiply what is there
  p.kblocks = (int)(g.k / 128);
  p.split = split;
  p.x_bf16 = (const __nv_bfloat16*)g.x_bf16;
  CUtensorMap map_x = {}, map_w;
  int rc = 0;
  if (QUANT) {
    p.stage_bytes = W_BYTES;
    p.stages = quant_stages<G>(GATED, p.token_tile, (int)ceil_div(p.kblocks, split));
  } else {
    p.stage_bytes = W_BYTES + p.token_bytes;
    p.stages = std::min(kMaxStages, (G::SMEM_BYTES - G::fixed_bytes(GATED)) / p.stage_bytes);
    rc = pair_map_tokens(&map_x, g.x, g.T, g.k, 1, p.token_tile);
  }
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)g.k, (cuuint64_t)(GATED ? 2 * g.n : g.n)};
  const cuuint64_t strides[1] = {(cuuint64_t)g.k};
  const cuuint32_t box[2] = {KBYTES, GATED ? 64 : 128};
  rc = encode_tensor_map(&map_w, g.w, 1, 2, dims, strides, box, true, "weights");
  if (rc) return rc;
  p.x_scale = g.x_scale;
  p.w_scale = g.w_scale;
  p.bias = g.bias;
  p.addend = (const __nv_bfloat16*)g.addend;
  p.out = g.out;
  p.out_scale = g.out_scale;
  p.T = g.T;
  p.n = g.n;
  p.activation = g.activation;
  p.early = g.behind_late_trigger;
  const int ctas = GATED ? 2 * split : split;
  launch_pdl_cluster(kernel, ctas, dim3((unsigned)(ceil_div<int64_t>(g.n, 128) * p.token_tiles * ctas)), dim3(G::THREADS), G::SMEM_BYTES, st, map_x,
                     map_w, p);
  return launch_status("fp8_linear_kernel");
}

}  // namespace

int run_linear(LinearParams p, bool gated, cudaStream_t st) {
  if (p.T <= 0) return FMOE_OK;
  Choice c = choose(p, gated);
  if (t_debug_choice.split > 0) {
    c = t_debug_choice;
    const int kblocks = (int)(p.k / 128);
    c.split = std::min(c.split, std::min(kblocks, c.pair ? kMaxPairSplit : kMaxSplit / (gated ? 2 : 1)));
    c.quant = c.quant && p.x_bf16 && can_quant(p.T, gated, ceil_div(kblocks, c.split));
  }
  if (p.x_bf16 && !c.quant) {
    const int rc = run_quant_tokens(p.x_bf16, p.T, p.k, p.xq, p.xq_scale, st);
    if (rc) return rc;
    p.x = p.xq;
    p.x_scale = p.xq_scale;
    p.behind_late_trigger = true;
  }
  if (c.pair) return run_linear_pair(p, gated, c.split, st);
  auto go = [&](auto gated_c, auto quant_c) {
    constexpr bool GATED = decltype(gated_c)::value, QUANT = decltype(quant_c)::value;
    if (p.T <= 16) return launch<Few, GATED, QUANT>(p, c.split, st);
    if (p.T <= 32) return launch<Some, GATED, QUANT>(p, c.split, st);
    if constexpr (QUANT) return launch<Half, GATED, QUANT>(p, c.split, st);
    else return p.T <= 64 ? launch<Half, GATED, QUANT>(p, c.split, st) : launch<Many, GATED, QUANT>(p, c.split, st);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (c.quant) return gated ? go(Yes{}, Yes{}) : go(No{}, Yes{});
  return gated ? go(Yes{}, No{}) : go(No{}, No{});
}

namespace {

int check_linear(const LinearParams& p, bool gated, const char* who) {
  FMOE_REQUIRE(p.T >= 0 && p.n >= 1 && p.k >= 1, "%s: bad sizes T=%lld n=%lld k=%lld", who, (long long)p.T, (long long)p.n, (long long)p.k);
  FMOE_REQUIRE(p.k % 128 == 0, "%s: the reduction length must be a multiple of 128 (got %lld)", who, (long long)p.k);
  FMOE_REQUIRE(p.n % (gated ? 128 : 8) == 0, "%s: the output width must be a multiple of %d (got %lld)", who, gated ? 128 : 8, (long long)p.n);
  FMOE_REQUIRE(p.T < (1ll << 30) && p.n < (1ll << 30) && p.k < (1ll << 30) &&
                   8 * ceil_div<int64_t>(p.n, 128) * ceil_div<int64_t>(std::max<int64_t>(p.T, 1), 64) < (1ll << 31),
               "%s: sizes T=%lld n=%lld k=%lld are too large", who, (long long)p.T, (long long)p.n, (long long)p.k);
  FMOE_REQUIRE(!gated || p.activation == FMOE_ACT_SILU || p.activation == FMOE_ACT_GELU, "%s: unknown activation %d", who, p.activation);
  return FMOE_OK;
}

int check_pointers(const LinearParams& p, bool gated, const char* who) {
  FMOE_REQUIRE(p.w && p.w_scale && p.out && (!gated || p.out_scale), "%s: null pointer", who);
  FMOE_REQUIRE(aligned16(p.w) && aligned16(p.out) && aligned16(p.bias) && aligned16(p.addend) &&
                   ((reinterpret_cast<uintptr_t>(p.w_scale) | reinterpret_cast<uintptr_t>(p.out_scale)) & 3u) == 0,
               "%s: misaligned pointer", who);
  return FMOE_OK;
}

// Workspace of a call: quantised rows [T, K] with their scales (bf16 input), the activation [T, I] with its scales (mlp)
struct Areas {
  int64_t xq = -1, xs = -1, h = -1, hs = -1, total = 0;
  Areas(const fmoe_fp8_args& a, bool mlp) {
    auto take = [&](int64_t bytes) {
      const int64_t at = total;
      total += (bytes + 255) & ~(int64_t)255;
      return at;
    };
    if (a.x_dtype == FMOE_BF16) {
      xq = take(a.T * a.K);
      xs = take(a.T * (a.K / 128) * 4);
    }
    if (mlp) {
      h = take(a.T * a.I);
      hs = take(a.T * (a.I / 128) * 4);
    }
  }
};

enum class Call { kLinear, kGateUp, kMlp };

// The sizes of a call, checked: `first` is the product that reads x, `down` (mlp) the second one.
int lay_out(const fmoe_fp8_args* a, Call call, const char* who, LinearParams* first, LinearParams* down) {
  if (!a) return fail(FMOE_ERR_INVALID_ARG, "%s: args is null", who);
  if (a->struct_size != sizeof(fmoe_fp8_args))
    return fail(FMOE_ERR_INVALID_ARG, "%s: fmoe_fp8_args.struct_size is %u, this library's struct has %zu bytes "
                "(binding built against another header?)", who, a->struct_size, sizeof(fmoe_fp8_args));
  FMOE_REQUIRE(a->x_dtype == FMOE_BF16 || a->x_dtype == FMOE_E4M3, "%s: x must be bf16 or e4m3", who);
  first->T = a->T;
  first->n = call == Call::kLinear ? a->N : a->I;
  first->k = a->K;
  first->activation = a->activation;
  int rc = check_linear(*first, call != Call::kLinear, who);
  if (rc || call != Call::kMlp) return rc;
  down->T = a->T;
  down->n = a->N;
  down->k = a->I;
  return check_linear(*down, false, who);
}

int run_call(const fmoe_fp8_args* a, Call call, const char* who, cudaStream_t st) {
  LinearParams first, down;
  int rc = lay_out(a, call, who, &first, &down);
  if (rc || a->T == 0) return rc;
  const Areas at(*a, call == Call::kMlp);
  FMOE_REQUIRE(call != Call::kGateUp || (!a->bias && !a->addend), "%s: bias and addend join the last product of a call", who);
  FMOE_REQUIRE(a->x && aligned16(a->x), "%s: x is null or misaligned", who);
  FMOE_REQUIRE(at.total == 0 || (a->workspace && (reinterpret_cast<uintptr_t>(a->workspace) & 255u) == 0 && a->workspace_bytes >= at.total),
               "%s: the workspace is null, not 256-byte aligned or too small (%lld bytes given, %lld needed)", who,
               (long long)a->workspace_bytes, (long long)at.total);
  uint8_t* ws = reinterpret_cast<uint8_t*>(a->workspace);
  first.w = a->w;
  first.w_scale = a->w_scale;
  LinearParams& last = call == Call::kMlp ? down : first;
  last.out = a->out;
  if (call != Call::kGateUp) {
    last.bias = a->bias;
    last.addend = a->addend;
  } else {
    first.out_scale = a->out_scale;
  }
  if (call == Call::kMlp) {
    first.out = ws + at.h;
    first.out_scale = reinterpret_cast<float*>(ws + at.hs);
    down.x = first.out;
    down.x_scale = first.out_scale;
    down.w = a->w2;
    down.w_scale = a->w2_scale;
    down.behind_late_trigger = true;
  }
  rc = check_pointers(first, call != Call::kLinear, who);
  if (!rc && call == Call::kMlp) rc = check_pointers(down, false, who);
  if (rc) return rc;
  if (a->x_dtype == FMOE_BF16) {
    first.x_bf16 = a->x;
    first.xq = ws + at.xq;
    first.xq_scale = reinterpret_cast<float*>(ws + at.xs);
  } else {
    FMOE_REQUIRE(a->x_scale && (reinterpret_cast<uintptr_t>(a->x_scale) & 3u) == 0, "%s: e4m3 rows need x_scale", who);
    first.x = a->x;
    first.x_scale = a->x_scale;
  }
  rc = run_linear(first, call != Call::kLinear, st);
  if (rc || call != Call::kMlp) return rc;
  return run_linear(down, false, st);
}

int64_t workspace_bytes(const fmoe_fp8_args* a, Call call, const char* who) {
  LinearParams first, down;
  if (lay_out(a, call, who, &first, &down)) return -1;
  return Areas(*a, call == Call::kMlp).total;
}

}  // namespace

void debug_linear_choice(int kernel, int split) { t_debug_choice = {kernel == 1, split, kernel == 2}; }

int status_word_linear_pair(int* out, bool clear);

// of both kernels
int status_word_linear(int* out, bool clear) {
  int zero = 0;
  int pair = 0;
  const int rc = status_word_linear_pair(&pair, clear);
  if (rc) return rc;
  FMOE_CUDA_OK(cudaMemcpyFromSymbol(out, g_device_status_linear, sizeof(int)));
  if (clear && *out != 0) FMOE_CUDA_OK(cudaMemcpyToSymbol(g_device_status_linear, &zero, sizeof(int)));
  if (*out == 0) *out = pair;
  return FMOE_OK;
}

}  // namespace fmoe

extern "C" int64_t fmoe_fp8_linear_workspace_bytes(const fmoe_fp8_args* args) {
  return fmoe::workspace_bytes(args, fmoe::Call::kLinear, "fp8_linear");
}
extern "C" int fmoe_fp8_linear(const fmoe_fp8_args* args, void* stream) {
  return fmoe::run_call(args, fmoe::Call::kLinear, "fp8_linear", (cudaStream_t)stream);
}
extern "C" int64_t fmoe_fp8_gate_up_workspace_bytes(const fmoe_fp8_args* args) {
  return fmoe::workspace_bytes(args, fmoe::Call::kGateUp, "fp8_gate_up");
}
extern "C" int fmoe_fp8_gate_up(const fmoe_fp8_args* args, void* stream) {
  return fmoe::run_call(args, fmoe::Call::kGateUp, "fp8_gate_up", (cudaStream_t)stream);
}
extern "C" int64_t fmoe_fp8_mlp_workspace_bytes(const fmoe_fp8_args* args) {
  return fmoe::workspace_bytes(args, fmoe::Call::kMlp, "fp8_mlp");
}
extern "C" int fmoe_fp8_mlp(const fmoe_fp8_args* args, void* stream) {
  return fmoe::run_call(args, fmoe::Call::kMlp, "fp8_mlp", (cudaStream_t)stream);
}
extern "C" int fmoe_debug_linear_kernel(int kernel, int split) {
  FMOE_REQUIRE(kernel >= 0 && kernel <= 2 && split >= 0 && split <= fmoe::kMaxSplit, "debug_linear_kernel: kernel %d, split %d", kernel, split);
  fmoe::debug_linear_choice(kernel, split);
  return FMOE_OK;
}
