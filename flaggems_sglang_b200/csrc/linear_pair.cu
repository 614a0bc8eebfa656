// Dense e4m3 products with block scales for many tokens (linear.cuh): persistent CTA pairs (cta_group::2).
//
//   tile      : 256 tokens on M (128 in each CTA) x 256 weight rows on N in two halves: 128 channels each, or (gate/up) 64 gate rows and
//               the same 64 up rows; a CTA loads 64 rows of either.  A thread of the fold owns one token: its activation scale is one
//               value per K block, and the weight scale one value per 128 rows
//   K block   : 128 bytes per row; for each half 4 MMAs of 256 x 128 x 32 into a fresh TMEM partial of 128 columns, of which there are four
//   warps 0-7 : fold + epilogue.  Warp w: TMEM lanes 32 * (w % 4).., half w / 4: 128 sums per thread, and 64 further registers for the
//               columns on their way: each 32 are replaced by the next as soon as they have been added, and the partial is handed back
//               before the last 64 are.  The two halves' warps run half a K block apart, so that one's reads and waits are beside the
//               other's FMAs
//   warp 8     : TMA of tokens and weights     warp 10: MMA (CTA 0)     warp 11: scales, eight K blocks at a time, transposed into a ring
//   warp 9     : the addend into 64 KB of shared memory while the tile is multiplied, and the output from there, both by TMA.  The fold adds
//                and rounds in place, so that a tile's stores run beside the next one's MMAs: with each warp's loads and stores from its
//                registers 4096 x 2048 x 7168 with an addend took 91 us, this way 64; 8192 x 7168 x 4096 209 -> 193.  The ring gives up
//                two of six stages for it, which costs nothing.
// SPLIT: up to four pairs of a cluster share a tile's K blocks; their sums meet through distributed shared memory as in linear.cu.
// What bounds it: up to some 1500 tokens about 800 clocks per K block and tile, of which shared memory (32 KB in, 48 KB of operands at 128
// bytes per clock) needs 640 and what an SM takes in from L2 655; from there on the power limit (8192 x 7168 x 4096: 193 us, 2.5 PFLOP/s
// at about 1.5 GHz).  Tried: one MMA over all 256 rows of N (512 clocks of shared memory, but only two partials for the fold's round
// trip: the same at 8192 tokens, 2048 x 2048 x 7168 42 us against 38); reads of the next K block before the last of this one are added
// (30.5 us against 28.4 for one round of K = 7168); 16 fold warps of 64 sums (223 us against 210 at 8192 tokens), packed FMAs (242), waits
// that poll without a hint (251).  An arrival behind a branch left the fold's warps split, so that each FMA was issued twice: 247 us where
// it then took 217.
#include "linear.cuh"
#include "pair.cuh"
#include "rows.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace fmoe {

// This translation unit's status word; read by status_word_linear_pair().
__device__ int g_device_status_linear_pair = 0;

namespace {

constexpr int KBYTES = 128;
constexpr int HALF_BYTES = 128 * KBYTES;          // this CTA's tokens, or weight rows, of a stage
constexpr int STAGE_BYTES = 2 * HALF_BYTES;
constexpr int STAGES = 4;
constexpr int kFoldWarps = 8;
constexpr int kThreads = (kFoldWarps + 4) * 32;
constexpr int kFoldRegs = 216, kOtherRegs = 72;   // together the launch's 384 x 168
constexpr int kGroup = 8;                         // K blocks per slot of scales
constexpr int kSlots = 3;
constexpr int SLOT_FLOATS = kGroup * (128 + 2);   // [K block][token], [K block][weight block]
constexpr int BAR_BYTES = 512;
constexpr int SUM_PITCH = 260;                    // floats from token to token: 16-byte accesses of eight lanes take all banks
constexpr int kMaxSplit = kMaxPairSplit;
constexpr int AMAX_FLOATS = 2 * 2 * 128;          // [tile parity][column half][token]
constexpr int OUT_BOX = 32 * 128;                  // 32 tokens x 64 channels on their way out, rows of 128 bytes swizzled as TMA has them
constexpr int OUT_BYTES = kFoldWarps * 2 * OUT_BOX;
constexpr int STRIP_PITCH = 80;                    // gated: bytes from token to token of a fold warp's strip: 64 and a shift of banks
constexpr int STRIP_BYTES = 32 * STRIP_PITCH;
constexpr int kSmemUsed = STAGES * STAGE_BYTES + OUT_BYTES + BAR_BYTES + (kSlots * SLOT_FLOATS + AMAX_FLOATS) * 4;
// All of an SM's: a CTA of another kernel that fitted beside and had TMEM would wait here for this one's end (512 columns), while its cluster
// waits for it, or this one for that one's.
constexpr int kSmemBytes = 227 * 1024;
static_assert(kSmemUsed <= kSmemBytes, "shared memory");
static_assert(128 * SUM_PITCH * 4 <= STAGES * STAGE_BYTES + OUT_BYTES && STRIP_BYTES <= 2 * OUT_BOX, "sums, strips");

struct KernelParams {
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  const __nv_bfloat16* addend;
  void* out;
  float* out_scale;
  int64_t n;
  int T, kblocks, w_blocks;        // w_blocks: 128-row blocks of the weights
  int token_tiles, w_tiles, group;  // group: token tiles that run beside one another
  int activation;
  int early;
  int split;
};

__device__ __forceinline__ void report(int code) { atomicCAS(&g_device_status_linear_pair, 0, code); }
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity));
}

// Stays between the TMEM reads and waits that it is written between.
__device__ __forceinline__ void fma_in_place(float& acc, float v, float f) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc) : "f"(v), "f"(f));
}

// Tile `i`: groups of token tiles, inside a group the token tile varies fastest, so that the tiles that run at the same time share
// weight rows through L2 and the group's token rows stay hot.
struct Tile {
  int token, w;
  __device__ __forceinline__ Tile(int i, const KernelParams& p) {
    const int per_group = p.group * p.w_tiles, g = i / per_group, r = i - g * per_group;
    const int in_group = min(p.group, p.token_tiles - g * p.group);
    w = r / in_group;
    token = g * p.group + r - w * in_group;
  }
};

// SPLIT: a tile per cluster of `split` pairs, each with a part of its K blocks
template <bool GATED, bool MOVE, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
fp8_linear_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_addend, const KernelParams p) {
  constexpr bool BOXES = !GATED && !SPLIT;  // the output leaves by TMA
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* outgoing = smem + STAGES * STAGE_BYTES;  // [fold warp][64 channels][token]
  uint64_t* bars = reinterpret_cast<uint64_t*>(outgoing + OUT_BYTES);
  uint64_t* full_bar = bars;                // [STAGES] used in CTA 0: both CTAs' loads -> MMA
  uint64_t* empty_bar = bars + STAGES;      // [STAGES] per CTA: MMA -> TMA
  uint64_t* part_full = bars + 2 * STAGES;  // [4] per CTA: MMA -> fold; 2 * (K block % 2) + half
  uint64_t* part_empty = part_full + 4;     // [4] used in CTA 0: folds of both CTAs -> MMA
  uint64_t* sc_full = part_empty + 4;       // [kSlots]
  uint64_t* sc_empty = sc_full + kSlots;    // [kSlots]
  uint64_t* amax_bar = sc_empty + kSlots;   // [4] the two warps that hold a token's 128 channels
  uint64_t* out_ready = amax_bar + 4;       // [1] the boxes are free, and hold the tile's addend
  uint64_t* out_full = out_ready + 1;       // [kFoldWarps] a warp's boxes are complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(out_full + kFoldWarps);
  float* scales = reinterpret_cast<float*>(outgoing + OUT_BYTES + BAR_BYTES);
  float* amax_buf = scales + kSlots * SLOT_FLOATS;

  const int warp = ptx::uniform_warp_id(), lane = threadIdx.x & 31;
  const int cluster_rank = (int)ptx::cluster_ctarank(), rank = cluster_rank & 1;
  const int S = SPLIT ? p.split : 1;
  const int worker = blockIdx.x / (2 * S), workers = gridDim.x / (2 * S);
  const int tiles = p.token_tiles * p.w_tiles;
  const int kb0 = SPLIT ? p.kblocks * (cluster_rank >> 1) / S : 0, kb1 = SPLIT ? p.kblocks * ((cluster_rank >> 1) + 1) / S : p.kblocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 4; ++b) {
      ptx::mbar_init(&part_full[b], 1);
      ptx::mbar_init(&part_empty[b], kFoldWarps);  // the half's four warps of both CTAs
    }
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(&sc_full[s], 1);
      ptx::mbar_init(&sc_empty[s], kFoldWarps);
    }
    for (int q = 0; q < 4; ++q) ptx::mbar_init(&amax_bar[q], 2);
    ptx::mbar_init(out_ready, 1);
    for (int q = 0; q < kFoldWarps; ++q) ptx::mbar_init(&out_full[q], 1);
    ptx::fence_barrier_init();
  }
  if (warp == kFoldWarps && lane == 0) {
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_w);
    if (BOXES) ptx::prefetch_tensormap(&map_out);
  }
  if (warp == kFoldWarps + 2) {
    ptx::tmem_alloc_pair(tmem_slot, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (MOVE && warp >= kFoldWarps) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp < kFoldWarps) {
    // ---------------- fold + epilogue ----------------
    if constexpr (MOVE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFoldRegs));
    pdl_entry_late();
    const int quarter = warp & 3, piece = warp >> 2;
    const uint32_t from = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t empty0 = ptx::smem_u32(part_empty) & ~ptx::kPeerRankBit;
    uint32_t step = 0, sc_step = 0;  // K blocks folded so far; the same with whole slots of scales for every tile
    bool alive = true;
    int ltile = 0;
    for (int i = worker; i < tiles && alive; i += workers, ++ltile) {
      const Tile tl(i, p);
      float acc[128];
#pragma unroll
      for (int c = 0; c < 128; ++c) acc[c] = 0.f;
      const uint32_t end = step + (kb1 - kb0);
#pragma unroll 1
      for (; step != end; ++step, ++sc_step) {
        const uint32_t slot = sc_step / kGroup % kSlots;
        if (sc_step % kGroup == 0 && !warp_wait(&sc_full[slot], (sc_step / (kGroup * kSlots)) & 1)) {
          report(0x2400);
          alive = false;
          break;
        }
        const float* sc = scales + slot * SLOT_FLOATS;
        const float a = sc[(sc_step % kGroup) * 128 + quarter * 32 + lane];
        const float2 w = *reinterpret_cast<const float2*>(sc + kGroup * 128 + (sc_step % kGroup) * 2);
        const float f0 = a * (GATED ? w.x : (piece ? w.y : w.x)), f1 = GATED ? a * w.y : f0;
        const uint32_t buf = 2 * (step & 1) + piece;
        if (!warp_wait(&part_full[buf], (step >> 1) & 1)) {
          report(0x2440);
          alive = false;
          break;
        }
        ptx::tc_fence_after_sync();
        // two reads of 32 columns are in flight; each is replaced by the next as soon as it has been added
        uint32_t v[2][32];
        const uint32_t at = from + buf * 128;
        auto add = [&](auto c_c) {
          constexpr int c = decltype(c_c)::value;
#pragma unroll
          for (int j = 0; j < 32; ++j) fma_in_place(acc[32 * c + j], __uint_as_float(v[c & 1][j]), c < 2 ? f0 : f1);
        };
        ptx::tmem_ld_32x32b_x32(at, v[0]);
        ptx::tmem_ld_32x32b_x32(at + 32, v[1]);
        ptx::tmem_ld_wait();
        add(std::integral_constant<int, 0>{});
        ptx::tmem_ld_32x32b_x32(at + 64, v[0]);
        add(std::integral_constant<int, 1>{});
        ptx::tmem_ld_32x32b_x32(at + 96, v[1]);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        ptx::mbar_arrive_cluster_if(lane == 0, empty0 + 8 * buf);
        add(std::integral_constant<int, 2>{});
        add(std::integral_constant<int, 3>{});
        if (sc_step % kGroup == kGroup - 1) ptx::mbar_arrive_if(lane == 0, &sc_empty[slot]);
      }
      if (!alive) break;
      if constexpr (SPLIT) {
        // Sums to shared memory in place of the ring, [token][channel] (gate and up halves), once the last partials of both halves are
        // complete: every MMA has read its operands then.
        if (!warp_wait(&part_full[2 * ((step - 1) & 1) + (piece ^ 1)], ((step - 1) >> 1) & 1)) {
          report(0x2480);
          break;
        }
        float* sums = reinterpret_cast<float*>(smem) + (quarter * 32 + lane) * SUM_PITCH;
#pragma unroll
        for (int c = 0; c < 128; c += 4)
          *reinterpret_cast<float4*>(sums + (GATED ? (c < 64 ? 64 * piece + c : 64 + 64 * piece + c) : 128 * piece + c)) =
              make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        continue;
      }
      if (sc_step % kGroup != 0) {  // the tile's last slot is not full
        if (lane == 0) ptx::mbar_arrive(&sc_empty[sc_step / kGroup % kSlots]);
        sc_step += kGroup - sc_step % kGroup;
      }

      if constexpr (GATED) {
        // The warp's 32 tokens leave through its strip: lane l holds token l's values, and stores those of tokens l / 4 + 8 i, 16 bytes each.
        const int64_t t0 = (int64_t)tl.token * 256 + rank * 128 + quarter * 32;
        uint8_t* strip = outgoing + warp * STRIP_BYTES;
        uint4* own = reinterpret_cast<uint4*>(strip + lane * STRIP_PITCH);
        uint4* dealt = reinterpret_cast<uint4*>(strip + (lane >> 2) * STRIP_PITCH + (lane & 3) * 16);  // token lane / 4 + 8 i: 8 i rows on
        constexpr int kDealtStep = 8 * STRIP_PITCH / 16;
        const int mine = (int)min((int64_t)32, p.T - t0) - (lane >> 2);  // of the four tokens, those with 8 i < mine are there
        float amax = 0.f;
        auto activate = [&](auto activation) {
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            acc[j] = act_mul_fast(acc[j], acc[64 + j], decltype(activation)::value);
            amax = fmaxf(amax, fabsf(acc[j]));
          }
        };
        if (p.activation == FMOE_ACT_GELU) activate(std::integral_constant<int, FMOE_ACT_GELU>{});
        else activate(std::integral_constant<int, FMOE_ACT_SILU>{});
        // the tile's 128 channels of a token are one quantisation group, held by two warps
        float* am = amax_buf + (ltile & 1) * 256 + quarter * 32 + lane;
        am[128 * piece] = amax;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&amax_bar[quarter]);
        if (!warp_wait(&amax_bar[quarter], ltile & 1)) {
          report(0x24c0);
          break;
        }
        amax = fmaxf(amax, am[128 * (piece ^ 1)]);
        const float s = group_scale(amax), r = __frcp_rn(s);
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t word[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float v4[4] = {acc[c + 4 * q], acc[c + 4 * q + 1], acc[c + 4 * q + 2], acc[c + 4 * q + 3]};
            word[q] = quant4(v4, s, r, amax <= 3.0e38f);
          }
          own[c / 16] = make_uint4(word[0], word[1], word[2], word[3]);
        }
        if (piece == 0 && t0 + lane < p.T) p.out_scale[(t0 + lane) * (p.n / 128) + tl.w] = s;
        __syncwarp();
        uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + (t0 + (lane >> 2)) * p.n + tl.w * 128 + piece * 64 + (lane & 3) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (8 * i < mine) *reinterpret_cast<uint4*>(dst + 8 * i * p.n) = dealt[i * kDealtStep];
        __syncwarp();
      } else {
        // Into the warp's two boxes, which hold the addend's values so far, and on by TMA: the stores run beside the next tile.
        if (!warp_wait(out_ready, ltile & 1)) {
          report(0x2500);
          break;
        }
        const int64_t ch0 = (int64_t)tl.w * 256 + piece * 128;
        uint8_t* row = outgoing + warp * 2 * OUT_BOX + lane * 128;
#pragma unroll
        for (int c = 0; c < 128; c += 8) {
          uint4* at = reinterpret_cast<uint4*>(row + c / 64 * OUT_BOX + ((c / 8 % 8 ^ (lane & 7)) << 4));
          if (p.bias && ch0 + c < p.n) {
            const float4 b0 = __ldg(reinterpret_cast<const float4*>(p.bias + ch0 + c)), b1 = __ldg(reinterpret_cast<const float4*>(p.bias + ch0 + c) + 1);
            acc[c] += b0.x;
            acc[c + 1] += b0.y;
            acc[c + 2] += b0.z;
            acc[c + 3] += b0.w;
            acc[c + 4] += b1.x;
            acc[c + 5] += b1.y;
            acc[c + 6] += b1.z;
            acc[c + 7] += b1.w;
          }
          if (p.addend) {
            const uint4 raw = *at;
            const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              acc[c + 2 * u] += __low2float(e[u]);
              acc[c + 2 * u + 1] += __high2float(e[u]);
            }
          }
          *at = make_uint4(pack_bf16x2(acc[c], acc[c + 1]), pack_bf16x2(acc[c + 2], acc[c + 3]), pack_bf16x2(acc[c + 4], acc[c + 5]),
                           pack_bf16x2(acc[c + 6], acc[c + 7]));
        }
        ptx::fence_proxy_async();
        __syncwarp();
        ptx::mbar_arrive_if(lane == 0, &out_full[warp]);
      }
    }
  } else if (warp == kFoldWarps) {
    // ---------------- TMA: this CTA's half of the tile's tokens, and its 128 weight rows ----------------
    if (ptx::elect_one()) {
      const uint32_t ring = ptx::smem_u32(smem), bar_full0 = ptx::smem_u32(full_bar) & ~ptx::kPeerRankBit;
      auto load_weights = [&](const Tile& tl, int kb, int s) {
        // 64 rows for each half: 64 channels from here, or the same 64 channels' gate rows (CTA 0) and up rows
        const int row = GATED ? tl.w * 128 + rank * (int)p.n : tl.w * 256 + rank * 64;
        const uint32_t bar = bar_full0 + s * 8, dst = ring + s * STAGE_BYTES + HALF_BYTES;
        ptx::tma_load_2d_pair(dst, &map_w, kb * KBYTES, row, bar);
        ptx::tma_load_2d_pair(dst + HALF_BYTES / 2, &map_w, kb * KBYTES, row + (GATED ? 64 : 128), bar);
      };
      int stage = 0, ahead = 0;
      uint32_t phase = 0;
      bool alive = true;
      if (p.early) {  // weights that nothing before this kernel writes are on their way before the tokens are there
        const Tile tl(worker, p);
        for (ahead = 0; ahead < min(STAGES, kb1 - kb0); ++ahead) load_weights(tl, kb0 + ahead, ahead);
      }
      pdl_wait();
      pdl_trigger();
      for (int i = worker; i < tiles && alive; i += workers) {
        const Tile tl(i, p);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1)) {
            report(0x2100 | stage);
            alive = false;
            break;
          }
          if (rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[stage], 2 * STAGE_BYTES);
          ptx::tma_load_2d_pair(ring + stage * STAGE_BYTES, &map_x, kb * KBYTES, tl.token * 256 + rank * 128, bar_full0 + stage * 8);
          if (ahead > 0) --ahead;
          else load_weights(tl, kb, stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      for (int s = 0; alive && s < STAGES; ++s) {  // nothing is in flight when this CTA ends
        if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1)) {
          report(0x2180 | stage);
          break;
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == kFoldWarps + 1) {
    // ---------------- addend and output of a tile, by TMA ----------------
    if (BOXES && ptx::elect_one()) {
      pdl_wait();
      const uint32_t boxes = ptx::smem_u32(outgoing);
      bool alive = true;
      int ltile = 0;
      for (int i = worker; i < tiles && alive; i += workers, ++ltile) {
        const Tile tl(i, p);
        const int t0 = tl.token * 256 + rank * 128, ch0 = tl.w * 256;
        const int quarters = p.T > t0 ? min(4, (p.T - t0 + 31) / 32) : 0, cols = (int)min((int64_t)4, (p.n - ch0 + 63) / 64);
        auto box = [&](int quarter, int c) { return boxes + ((c >> 1) * 8 + quarter * 2 + (c & 1)) * OUT_BOX; };
        ptx::tma_store_wait_read();
        if (p.addend) {
          ptx::mbar_arrive_expect_tx(out_ready, quarters * cols * OUT_BOX);
          for (int c = 0; c < cols; ++c)
            for (int q = 0; q < quarters; ++q) ptx::tma_load_2d(box(q, c), &map_addend, ch0 + 64 * c, t0 + 32 * q, ptx::smem_u32(out_ready));
        } else {
          ptx::mbar_arrive(out_ready);
        }
        if (!ptx::mbar_wait(out_ready, ltile & 1)) {  // and nothing is in flight when this CTA ends
          report(0x2540);
          break;
        }
        for (int w = 0; w < kFoldWarps && alive; ++w) {
          if (!ptx::mbar_wait_relaxed(&out_full[w], ltile & 1)) {
            report(0x2580 | w);
            alive = false;
          } else if ((w & 3) < quarters) {
            for (int c = w / 4 * 2; c < min(cols, w / 4 * 2 + 2); ++c) ptx::tma_store_2d(&map_out, box(w & 3, c), ch0 + 64 * c, t0 + 32 * (w & 3));
          }
        }
        ptx::tma_store_commit();
      }
      ptx::tma_store_wait();
    }
    __syncwarp();
  } else if (warp == kFoldWarps + 2) {
    // ---------------- MMA issuer (CTA 0): one fresh partial per K block ----------------
    if (rank == 0 && ptx::elect_one()) {
      pdl_wait();  // the limit of the waits below counts from here: a kernel ahead of this one may run on for any time
      const uint32_t ring = ptx::smem_u32(smem);
      const uint64_t da0 = ptx::smem_desc_sw128(ring), db0 = ptx::smem_desc_sw128(ring + HALF_BYTES);
      constexpr uint32_t idesc = ptx::make_idesc(/*e4m3*/ 0, 256, 128);
      const uint16_t pair_mask = (uint16_t)(3 << cluster_rank);
      int stage = 0;
      uint32_t phase = 0, step = 0;
      bool alive = true;
      for (int i = worker; i < tiles && alive; i += workers) {
        for (int kb = kb0; kb < kb1; ++kb, ++step) {
          if (!ptx::mbar_wait(&full_bar[stage], phase)) {
            report(0x2200 | stage);
            alive = false;
            break;
          }
          const uint64_t off = (uint64_t)(stage * (STAGE_BYTES >> 4));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t buf = 2 * (step & 1) + h;
            if (!ptx::mbar_wait(&part_empty[buf], ((step >> 1) & 1) ^ 1)) {
              report(0x2240 | buf);
              alive = false;
              break;
            }
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int kk = 0; kk < KBYTES / 32; ++kk)
              ptx::mma_f8f6f4_ss_pair(tmem_base + buf * 128, da0 + off + 2 * kk, db0 + off + h * (HALF_BYTES / 2 >> 4) + 2 * kk, idesc, kk != 0);
            ptx::mma_commit_both(&part_full[buf], pair_mask);
          }
          if (!alive) break;
          ptx::mma_commit_both(&empty_bar[stage], pair_mask);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- scales ----------------
    pdl_entry_late();
    uint32_t group = 0;
    bool alive = true;
    const bool vec = p.kblocks % 4 == 0 && kb0 % 4 == 0 && (reinterpret_cast<uintptr_t>(p.x_scale) & 15) == 0;
    for (int i = worker; i < tiles && alive; i += workers) {
      const Tile tl(i, p);
      const int t0 = tl.token * 256 + rank * 128 + lane;
      const int b0 = GATED ? tl.w : 2 * tl.w, b1 = GATED ? tl.w + (int)(p.n / 128) : min(2 * tl.w + 1, p.w_blocks - 1);
      const float* w_mine = p.w_scale + (int64_t)(lane & 1 ? b1 : b0) * p.kblocks;  // lanes 0-15: K block lane / 2, block lane % 2
      if (!GATED && SPLIT && p.addend) {  // on its way to L2 while the tile is multiplied: all workers read theirs at about the same time
        const int64_t t = tl.token * 256 + rank * 128, ch = (int64_t)tl.w * 256;
        const int lines = (int)(min((int64_t)256, p.n - ch) * 2 + 127) / 128;
        for (int r = lane; r < 128 && t + r < p.T; r += 32)
          for (int l = 0; l < lines; ++l) prefetch_l2(reinterpret_cast<const uint8_t*>(p.addend + (t + r) * p.n + ch) + 128 * l);
      }
      for (int kb = kb0; kb < kb1; kb += kGroup, ++group) {
        const int slot = group % kSlots, count = min(kGroup, kb1 - kb);
        const float w = lane < 2 * count ? __ldg(w_mine + kb + (lane >> 1)) : 0.f;
        float* dst = scales + slot * SLOT_FLOATS;
#pragma unroll 1
        for (int q = 0; q < kGroup; q += 4) {  // four K blocks at a time: this warp has few registers
          float4 a[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float* src = p.x_scale + (int64_t)(t0 + 32 * j) * p.kblocks + kb + q;
            a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t0 + 32 * j < p.T && q < count) {
              if (vec) {
                a[j] = __ldg(reinterpret_cast<const float4*>(src));
              } else {
                a[j].x = __ldg(src);
                if (q + 1 < count) a[j].y = __ldg(src + 1);
                if (q + 2 < count) a[j].z = __ldg(src + 2);
                if (q + 3 < count) a[j].w = __ldg(src + 3);
              }
            }
          }
          if (q == 0 && !warp_wait(&sc_empty[slot], ((group / kSlots) & 1) ^ 1)) {
            report(0x2300 | slot);
            alive = false;
            break;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float* d = dst + q * 128 + 32 * j + lane;
            d[0] = a[j].x;
            d[128] = a[j].y;
            d[256] = a[j].z;
            d[384] = a[j].w;
          }
        }
        if (!alive) break;
        if (lane < 2 * kGroup) dst[kGroup * 128 + lane] = w;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sc_full[slot]);
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync_all();  // nobody signals into a CTA that has left, and both are done with TMEM; SPLIT: all sums are there
  if (warp == kFoldWarps + 2) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
  if constexpr (SPLIT) {
    // A warp per token, a CTA's tokens dealt to the CTAs that share them (every second of the cluster)
    const Tile tl(worker, p);
    const int64_t t0 = (int64_t)tl.token * 256 + rank * 128;
    const int tokens = (int)max((int64_t)0, min((int64_t)128, p.T - t0));
    // (the fold warps: the others have given their registers away)
    if (warp < kFoldWarps) {
      join_tokens<2, kMaxSplit>((cluster_rank >> 1) + S * warp, S * kFoldWarps, tokens, S, rank, 2, true, ptx::smem_u32(smem) + lane * 16,
                                SUM_PITCH * 4, 512, [&](int t, float(&v)[2][4]) {
        if constexpr (GATED) {
          store_gated(v, p.activation, reinterpret_cast<uint8_t*>(p.out) + (t0 + t) * p.n + tl.w * 128,
                      p.out_scale + (t0 + t) * (p.n / 128) + tl.w);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t ch = (int64_t)tl.w * 256 + 128 * h + 4 * lane;
            if (ch < p.n) store_plain(v[h], p.bias, p.addend, reinterpret_cast<__nv_bfloat16*>(p.out), (t0 + t) * p.n, ch);
          }
        }
      });
    }
    ptx::cluster_sync_relaxed();  // nobody leaves while its sums are read
  }
}

template <bool GATED, bool SPLIT>
int launch(const LinearParams& g, int split, cudaStream_t st) {
  auto kernel = fp8_linear_pair_kernel<GATED, true, SPLIT>;
  // setmaxnreg waits for good when the launch has fewer registers than the warps' shares add up to: a build that gives these threads
  // fewer than 168 gets the kernel without it
  static std::atomic<int> moves{-1};
  if (moves < 0) {
    cudaFuncAttributes fa;
    FMOE_CUDA_OK(cudaFuncGetAttributes(&fa, kernel));
    moves = fa.numRegs * kThreads >= (kFoldWarps * kFoldRegs + 4 * kOtherRegs) * 32;
  }
  if (!moves) kernel = fp8_linear_pair_kernel<GATED, false, SPLIT>;
  static PerDeviceOnce once_attr;
  const cudaError_t attr_err = per_device_once(once_attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  });
  if (attr_err != cudaSuccess) return fail(FMOE_ERR_CUDA, "set-up of the e4m3 pair kernel failed: %s", cudaGetErrorString(attr_err));
  const int64_t w_rows = GATED ? 2 * g.n : g.n;
  CUtensorMap map_x, map_w;
  int rc = pair_map_tokens(&map_x, g.x, g.T, g.k, 1, 128);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)g.k, (cuuint64_t)w_rows};
  const cuuint64_t strides[1] = {(cuuint64_t)g.k};
  const cuuint32_t box[2] = {KBYTES, 64};
  rc = encode_tensor_map(&map_w, g.w, 1, 2, dims, strides, box, true, "weights");
  if (rc) return rc;
  KernelParams p;
  p.x_scale = g.x_scale;
  p.w_scale = g.w_scale;
  p.bias = g.bias;
  p.addend = (const __nv_bfloat16*)g.addend;
  p.out = g.out;
  p.out_scale = g.out_scale;
  p.n = g.n;
  p.T = (int)g.T;
  p.kblocks = (int)(g.k / 128);
  p.w_blocks = (int)ceil_div<int64_t>(w_rows, 128);
  p.token_tiles = (int)ceil_div<int64_t>(g.T, 256);
  p.w_tiles = (int)ceil_div<int64_t>(g.n, GATED ? 128 : 256);
  p.group = pick_group_m(256, g.k);
  p.activation = g.activation;
  p.early = g.behind_late_trigger;
  p.split = split;
  const int64_t tiles = (int64_t)p.token_tiles * p.w_tiles;
  const int sms = device_sm_count();
  const int workers = (int)(SPLIT ? tiles : std::min<int64_t>((sms > 0 ? sms : 148) / 2, tiles));
  CUtensorMap map_out = {}, map_addend = {};
  if (!GATED && !SPLIT) {
    const cuuint64_t out_dims[2] = {(cuuint64_t)g.n, (cuuint64_t)g.T};
    const cuuint64_t out_strides[1] = {(cuuint64_t)g.n * 2};
    const cuuint32_t out_box[2] = {64, 32};
    rc = encode_tensor_map(&map_out, g.out, 2, 2, out_dims, out_strides, out_box, false, "output");
    if (!rc && g.addend) rc = encode_tensor_map(&map_addend, g.addend, 2, 2, out_dims, out_strides, out_box, false, "addend");
    if (rc) return rc;
  }
  launch_pdl_cluster(kernel, 2 * split, dim3(2 * split * workers), dim3(kThreads), kSmemBytes, st, map_x, map_w, map_out, map_addend, p);
  return launch_status("fp8_linear_pair_kernel");
}

}  // namespace

int run_linear_pair(const LinearParams& p, bool gated, int split, cudaStream_t st) {
  if (split > 1) return gated ? launch<true, true>(p, split, st) : launch<false, true>(p, split, st);
  return gated ? launch<true, false>(p, 1, st) : launch<false, false>(p, 1, st);
}

int status_word_linear_pair(int* out, bool clear) {
  int zero = 0;
  FMOE_CUDA_OK(cudaMemcpyFromSymbol(out, g_device_status_linear_pair, sizeof(int)));
  if (clear && *out != 0) FMOE_CUDA_OK(cudaMemcpyToSymbol(g_device_status_linear_pair, &zero, sizeof(int)));
  return FMOE_OK;
}

}  // namespace fmoe
