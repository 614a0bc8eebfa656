// Dense products of e4m3 operands with a scale per 128 channels of every token and per 128 x 128 block of the weights:
//     y[t, n] = sum_kb a[t, kb] * b[n / 128, kb] * (sum_{k in kb} xq[t, k] * wq[n, k])
// what a layer computes beside its routed experts (shared expert, attention projections).
//
// The tensor cores cannot apply a scale inside their accumulator that changes with K, so every K block of 128 is multiplied into
// a fresh TMEM partial (4 MMAs of K = 32) which the fold warps add, times a[t, kb] * b[n / 128, kb], to sums in registers.
//
//   tile    : 128 weight rows (gate/up: 128 gate rows and the same 128 up rows) on the MMA's M side x up to 64 or 128 tokens on N.
//             With the weights on M a call of one token costs a 16-column tile
//   split   : S CTAs of a cluster share a tile, each with a contiguous part of its K blocks, so that few tiles still fill the
//             chip.  Their sums meet through distributed shared memory, added in the order of the CTAs: the result does not
//             depend on timing, and there is no scratch in global memory and no counter
//   warps   : fold warps (four per 128 rows x 64 tokens: TMEM lane quarter = warp % 4, 64 sums per thread), then TMA, MMA, and
//             two that multiply token and weight scales into a ring of factors
//   epilogue: sums to shared memory [token][row], then a warp per token: a row of 128 channels is one coalesced store, and for
//             gate/up it is one quantisation group, whose largest magnitude is a warp reduction
// Every mbarrier wait is bounded; the cluster barriers are reached by every thread on every path.
#include "linear.cuh"
#include "pair.cuh"
#include "rows.cuh"

#include <algorithm>

namespace fmoe {

// This translation unit's status word; read by status_word_linear().
__device__ int g_device_status_linear = 0;

namespace {

constexpr int KBYTES = 128;
constexpr int W_BYTES = 128 * KBYTES;
constexpr int kMaxSmem = 227 * 1024;
constexpr int kMaxStages = 12;
constexpr int kGroup = 8;  // K blocks per factor slot
constexpr int kSlots = 4;
constexpr int BAR_BYTES = 512;

// HALVES: 1 = plain, 2 = gate rows and up rows; COLS: most tokens of a tile
template <int HALVES, int COLS>
struct Geo {
  static constexpr int FOLD_WARPS = 4 * HALVES * (COLS / 64);
  static constexpr int THREADS = (FOLD_WARPS + 4) * 32;
  static constexpr int BUF_COLS = HALVES * COLS;
  static constexpr int BUFS = 512 / BUF_COLS < 4 ? 512 / BUF_COLS : 4;
  static constexpr int TMEM_COLS = BUFS * BUF_COLS;
  static constexpr int KB_FLOATS = HALVES * COLS;  // factors of one K block
  static constexpr int SLOT_FLOATS = kGroup * KB_FLOATS;
  static constexpr int FIXED_BYTES = BAR_BYTES + kSlots * SLOT_FLOATS * 4;
  static constexpr int ROWS = 128 * HALVES;
  static constexpr int SUM_BYTES = COLS * ROWS * 4;  // the sums, in place of the ring
};

struct KernelParams {
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  const __nv_bfloat16* addend;
  void* out;
  float* out_scale;
  int64_t T, n;
  int kblocks;
  int token_tiles, token_tile;  // token_tile: a multiple of 16
  int stages, stage_bytes;
  int split;      // CTAs per tile
  int activation;
  int early;      // the weights are complete when the kernel starts
};

__device__ __forceinline__ void report(int code) { atomicCAS(&g_device_status_linear, 0, code); }

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity));
}

template <int HALVES, int COLS>
__global__ void __launch_bounds__(Geo<HALVES, COLS>::THREADS, 1)
fp8_linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const KernelParams p) {
  using G = Geo<HALVES, COLS>;
  extern __shared__ __align__(1024) uint8_t smem[];
  // barriers and factors first in the fixed part behind the ring; the ring itself starts at 0 (1024-byte aligned stages)
  uint8_t* fixed = smem + kMaxSmem - G::FIXED_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(fixed);
  uint64_t* full_bar = bars;                    // [stages] TMA -> MMA
  uint64_t* empty_bar = bars + kMaxStages;      // [stages] MMA -> TMA
  uint64_t* part_full = bars + 2 * kMaxStages;  // [BUFS] MMA -> fold
  uint64_t* part_empty = part_full + 4;         // [BUFS] fold -> MMA
  uint64_t* sc_full = part_empty + 4;           // [kSlots] factor warps -> fold
  uint64_t* sc_empty = sc_full + kSlots;        // [kSlots] fold -> factor warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + kSlots);
  float* factors = reinterpret_cast<float*>(fixed + BAR_BYTES);

  const int warp = ptx::uniform_warp_id(), lane = threadIdx.x & 31;
  const int S = p.split;
  const int rank = S > 1 ? (int)ptx::cluster_ctarank() : 0;
  const int tile = (int)blockIdx.x / S;
  const int row_tile = tile / p.token_tiles;
  const int tok0 = tile % p.token_tiles * p.token_tile;
  const int kb0 = (int)((int64_t)p.kblocks * rank / S), kb1 = (int)((int64_t)p.kblocks * (rank + 1) / S);
  const int up_tile = row_tile + (int)(p.n / 128);  // gate/up: the tile of up rows

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < G::BUFS; ++b) {
      ptx::mbar_init(&part_full[b], 1);
      ptx::mbar_init(&part_empty[b], G::FOLD_WARPS);
    }
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(&sc_full[s], 1);
      ptx::mbar_init(&sc_empty[s], G::FOLD_WARPS);
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
  const uint32_t tmem_base = *tmem_slot;

  if (warp == G::FOLD_WARPS) {
    // ---------------- TMA producer ----------------
    if (ptx::elect_one()) {
      const uint32_t ring = ptx::smem_u32(smem);
      const uint32_t bytes = HALVES * W_BYTES + p.token_tile * KBYTES;
      auto load_weights = [&](int kb, int s) {
        const uint32_t dst = ring + s * p.stage_bytes, bar = ptx::smem_u32(&full_bar[s]);
        ptx::mbar_arrive_expect_tx(&full_bar[s], bytes);
        ptx::tma_load_2d(dst, &map_w, kb * KBYTES, row_tile * 128, bar);
        if constexpr (HALVES == 2) ptx::tma_load_2d(dst + W_BYTES, &map_w, kb * KBYTES, up_tile * 128, bar);
      };
      auto load_tokens = [&](int kb, int s) {
        ptx::tma_load_2d(ring + s * p.stage_bytes + HALVES * W_BYTES, &map_x, kb * KBYTES, tok0, ptx::smem_u32(&full_bar[s]));
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
      const uint64_t dw0 = ptx::smem_desc_sw128(ring), dx0 = ptx::smem_desc_sw128(ring + HALVES * W_BYTES);
      const uint32_t idesc = ptx::make_idesc(/*e4m3*/ 0, 128, (uint32_t)p.token_tile);
      int stage = 0;
      uint32_t phase = 0;
      for (int step = 0; step < kb1 - kb0; ++step) {
        const int buf = step % G::BUFS;
        if (!ptx::mbar_wait(&full_bar[stage], phase)) {
          report(0x1200 | stage);
          break;
        }
        if (!ptx::mbar_wait(&part_empty[buf], ((step / G::BUFS) & 1) ^ 1)) {
          report(0x1240 | buf);
          break;
        }
        ptx::tc_fence_after_sync();
        const uint64_t off = (uint64_t)(stage * (p.stage_bytes >> 4));
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int kk = 0; kk < KBYTES / 32; ++kk)
            ptx::mma_f8f6f4_ss(tmem_base + buf * G::BUF_COLS + h * COLS, dw0 + off + h * (W_BYTES >> 4) + 2 * kk, dx0 + off + 2 * kk,
                               idesc, kk != 0);
        }
        ptx::mma_commit(&part_full[buf]);
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
    for (int g = me; g * kGroup < kb1 - kb0; g += 2) {
      const int first = kb0 + g * kGroup, count = min(kGroup, kb1 - first), slot = g % kSlots;
      float a[COLS / 32][kGroup];
#pragma unroll
      for (int j = 0; j < COLS / 32; ++j) {
        const int64_t t = tok0 + lane + 32 * j;
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          a[j][i] = (lane + 32 * j < p.token_tile && t < p.T && i < count) ? __ldg(p.x_scale + t * p.kblocks + first + i) : 0.f;
      }
      if (!warp_wait(&sc_empty[slot], ((g / kSlots) & 1) ^ 1)) {
        report(0x1300 | slot);
        break;
      }
      float* dst = factors + slot * G::SLOT_FLOATS + lane;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        if (i < count) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const float b = __ldg(p.w_scale + (int64_t)(h ? up_tile : row_tile) * p.kblocks + first + i);
#pragma unroll
            for (int j = 0; j < COLS / 32; ++j) dst[(i * HALVES + h) * COLS + 32 * j] = a[j][i] * b;
          }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sc_full[slot]);
    }
  } else {
    // ---------------- fold ----------------
    pdl_entry_late();
    const int piece = warp >> 2, half = piece / (COLS / 64), col0 = piece % (COLS / 64) * 64;
    const int cols = min(64, p.token_tile - col0);  // a multiple of 16, or nothing
    const uint32_t from = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + half * COLS + col0;
    float acc[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i] = 0.f;
    const int steps = kb1 - kb0;
    for (int step = 0; step < steps; ++step) {
      const int buf = step % G::BUFS, g = step / kGroup, slot = g % kSlots;
      if (step % kGroup == 0 && !warp_wait(&sc_full[slot], (g / kSlots) & 1)) {
        report(0x1400 | slot);
        break;
      }
      if (!warp_wait(&part_full[buf], (step / G::BUFS) & 1)) {
        report(0x1440 | buf);
        break;
      }
      ptx::tc_fence_after_sync();
      const float4* f4 = reinterpret_cast<const float4*>(factors + slot * G::SLOT_FLOATS + ((step % kGroup) * HALVES + half) * COLS + col0);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (16 * c < cols) {
          uint32_t v[16];
          ptx::tmem_ld_32x32b_x16(from + buf * G::BUF_COLS + 16 * c, v);
          float4 f[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) f[q] = f4[4 * c + q];
          ptx::tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            acc[16 * c + 4 * q] = fmaf(__uint_as_float(v[4 * q]), f[q].x, acc[16 * c + 4 * q]);
            acc[16 * c + 4 * q + 1] = fmaf(__uint_as_float(v[4 * q + 1]), f[q].y, acc[16 * c + 4 * q + 1]);
            acc[16 * c + 4 * q + 2] = fmaf(__uint_as_float(v[4 * q + 2]), f[q].z, acc[16 * c + 4 * q + 2]);
            acc[16 * c + 4 * q + 3] = fmaf(__uint_as_float(v[4 * q + 3]), f[q].w, acc[16 * c + 4 * q + 3]);
          }
        }
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(&part_empty[buf]);
        if (step % kGroup == kGroup - 1 || step == steps - 1) ptx::mbar_arrive(&sc_empty[slot]);
      }
    }
    // Sums to shared memory in place of the ring: the last partial is complete, so every MMA has read its operands.  A warp
    // writes 32 consecutive rows of a token.
    float* sums = reinterpret_cast<float*>(smem) + half * 128 + (warp & 3) * 32 + lane;
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (i < cols) sums[(col0 + i) * G::ROWS] = acc[i];
  }

  ptx::tc_fence_before_sync();
  if (S > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp == G::FOLD_WARPS + 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, G::TMEM_COLS);
  }

  // ---------------- epilogue: a warp per token, the tile's tokens dealt to the CTAs of the cluster ----------------
  const int tokens = (int)min((int64_t)p.token_tile, p.T - tok0);
  const uint32_t sums = ptx::smem_u32(smem) + lane * 16;
  for (int t = rank + S * warp; t < tokens; t += S * (G::THREADS / 32)) {
    float4 v[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) v[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const uint32_t at = sums + (t * G::ROWS + h * 128) * 4;
        const float4 part = ptx::ld_cluster_f4(S > 1 ? ptx::mapa(at, s) : at);
        v[h].x += part.x;
        v[h].y += part.y;
        v[h].z += part.z;
        v[h].w += part.w;
      }
    }
    const int64_t row = tok0 + t;
    const int64_t ch = (int64_t)row_tile * 128 + lane * 4;
    if constexpr (HALVES == 1) {
      if (ch < p.n) {
        if (p.bias) {
          const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + ch));
          v[0].x += b.x;
          v[0].y += b.y;
          v[0].z += b.z;
          v[0].w += b.w;
        }
        if (p.addend) {
          const uint2 raw = __ldg(reinterpret_cast<const uint2*>(p.addend + row * p.n + ch));
          const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw);
          v[0].x += __low2float(e[0]);
          v[0].y += __high2float(e[0]);
          v[0].z += __low2float(e[1]);
          v[0].w += __high2float(e[1]);
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + row * p.n + ch) =
            make_uint2(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[0].z, v[0].w));
      }
    } else {
      float h[4];
      h[0] = act_mul_fast(v[0].x, v[1].x, p.activation);
      h[1] = act_mul_fast(v[0].y, v[1].y, p.activation);
      h[2] = act_mul_fast(v[0].z, v[1].z, p.activation);
      h[3] = act_mul_fast(v[0].w, v[1].w, p.activation);
      float amax = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      const float s = group_scale(amax);
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + row * p.n + ch) = quant4(h, s, __frcp_rn(s), amax <= 3.0e38f);
      if (lane == 0) p.out_scale[row * (p.n / 128) + row_tile] = s;
    }
  }
  if (S > 1) ptx::cluster_sync_all();  // nobody leaves while its sums are read
}

// CTAs that share a tile's K blocks.  The time of a launch as a model: rounds of CTAs, each with a fixed part (launch, first
// loads, sums) and its K blocks at the slowest of HBM's share, what one SM takes in from L2, and the fold.
int pick_split(int64_t tiles, int kblocks, int halves, int cols, int sms) {
  int best = 1;
  double best_us = 1e30;
  for (int s = 1; s <= 8 && s <= kblocks; ++s) {
    const double ctas = (double)tiles * s, rounds = (double)ceil_div<int64_t>(tiles * s, sms);
    const double active = ctas < sms ? ctas : sms;
    const double hbm = active * halves * W_BYTES / 6.5e6, l2 = (halves * W_BYTES + cols * KBYTES) / 1.0e5;
    const double fold = (cols <= 64 ? 0.16 : 0.27) * halves;
    const double per_block = std::max(hbm, std::max(l2, fold));
    const double us = rounds * (ceil_div(kblocks, s) * per_block + 2.0 + (s > 1 ? 0.5 + 0.1 * s : 0.0));
    if (us < best_us) {
      best_us = us;
      best = s;
    }
  }
  return best;
}

template <int HALVES, int COLS>
int launch(const LinearParams& g, cudaStream_t st) {
  using G = Geo<HALVES, COLS>;
  static_assert(G::SUM_BYTES <= kMaxSmem - G::FIXED_BYTES, "shared memory");
  auto kernel = fp8_linear_kernel<HALVES, COLS>;
  static PerDeviceOnce once_attr;
  const cudaError_t attr_err = per_device_once(once_attr, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  });
  if (attr_err != cudaSuccess) return fail(FMOE_ERR_CUDA, "set-up of the e4m3 linear kernel failed: %s", cudaGetErrorString(attr_err));
  KernelParams p;
  p.token_tiles = (int)ceil_div<int64_t>(g.T, COLS);
  p.token_tile = (int)(ceil_div<int64_t>(ceil_div<int64_t>(g.T, p.token_tiles), 16) * 16);
  p.stage_bytes = HALVES * W_BYTES + p.token_tile * KBYTES;
  p.stages = std::min(kMaxStages, (kMaxSmem - G::FIXED_BYTES) / p.stage_bytes);
  p.kblocks = (int)(g.k / 128);
  const int64_t row_tiles = ceil_div<int64_t>(g.n, 128);
  const int sms = device_sm_count();
  p.split = pick_split(row_tiles * p.token_tiles, p.kblocks, HALVES, p.token_tile, sms > 0 ? sms : 148);
  const int64_t w_rows = HALVES * g.n;
  CUtensorMap map_x, map_w;
  int rc = pair_map_tokens(&map_x, g.x, g.T, g.k, 1, p.token_tile);
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)g.k, (cuuint64_t)w_rows};
  const cuuint64_t strides[1] = {(cuuint64_t)g.k};
  const cuuint32_t box[2] = {KBYTES, 128};
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
  launch_pdl_cluster(kernel, p.split, dim3((unsigned)(row_tiles * p.token_tiles * p.split)), dim3(G::THREADS), kMaxSmem, st, map_x, map_w, p);
  return launch_status("fp8_linear_kernel");
}

}  // namespace

int run_linear(const LinearParams& p, bool gated, cudaStream_t st) {
  if (p.T <= 0) return FMOE_OK;
  if (gated) return p.T <= 64 ? launch<2, 64>(p, st) : launch<2, 128>(p, st);
  return p.T <= 64 ? launch<1, 64>(p, st) : launch<1, 128>(p, st);
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
    first.x = ws + at.xq;
    first.x_scale = reinterpret_cast<float*>(ws + at.xs);
    first.behind_late_trigger = true;
    rc = run_quant_tokens(a->x, a->T, a->K, ws + at.xq, reinterpret_cast<float*>(ws + at.xs), st);
    if (rc) return rc;
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

int status_word_linear(int* out, bool clear) {
  int zero = 0;
  FMOE_CUDA_OK(cudaMemcpyFromSymbol(out, g_device_status_linear, sizeof(int)));
  if (clear && *out != 0) FMOE_CUDA_OK(cudaMemcpyToSymbol(g_device_status_linear, &zero, sizeof(int)));
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
