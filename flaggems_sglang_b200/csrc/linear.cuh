// Internal interface of the dense e4m3 products (linear.cu).
#pragma once
#include "gemm.cuh"
#include "ptx_sm100.cuh"
#include "rows.cuh"

#include <type_traits>

namespace fmoe {

// One product of e4m3 rows with e4m3 weights.  gated: `w` has 2n rows (gate rows, then up rows), the output is the quantised
// activation [T, n]; otherwise n rows, the output is bf16 [T, n].
struct LinearParams {
  int64_t T = 0, n = 0, k = 0;
  const void* x = nullptr;         // [T, k] e4m3
  const float* x_scale = nullptr;  // [T, k/128]
  const void* x_bf16 = nullptr;    // [T, k] instead of x and x_scale, quantised on the way: in the kernel, or to `xq` and `xq_scale` before it
  void* xq = nullptr;
  float* xq_scale = nullptr;
  const void* w = nullptr;
  const float* w_scale = nullptr;  // [ceil(rows/128), k/128]
  const float* bias = nullptr;     // [n]
  const void* addend = nullptr;    // bf16 [T, n]
  void* out = nullptr;
  float* out_scale = nullptr;      // gated: [T, n/128]
  int activation = FMOE_ACT_SILU;
  bool behind_late_trigger = false;  // the launch before is one of this library's that lets this one start only after its own
                                     // wait: the weights are complete when this kernel starts
};
constexpr int kMaxPairSplit = 4;  // pairs that share a tile there
int run_linear_pair(const LinearParams& p, bool gated, int split, cudaStream_t st);  // linear_pair.cu: many tokens
int run_linear(LinearParams p, bool gated, cudaStream_t st);

#if defined(__CUDACC__)
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// A warp stores 128 channels of a token, four of each lane from `ch` on: bias and addend join, one rounding.
__device__ __forceinline__ void store_plain(float (&v)[4], const float* bias, const __nv_bfloat16* addend, __nv_bfloat16* out, int64_t row_at,
                                            int64_t ch) {
  if (bias) {
    const float4 b = __ldg(reinterpret_cast<const float4*>(bias + ch));
    v[0] += b.x;
    v[1] += b.y;
    v[2] += b.z;
    v[3] += b.w;
  }
  if (addend) {  // may be `out` itself: no read-only path
    const uint2 raw = *reinterpret_cast<const uint2*>(addend + row_at + ch);
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw);
    v[0] += __low2float(e[0]);
    v[1] += __high2float(e[0]);
    v[2] += __low2float(e[1]);
    v[3] += __high2float(e[1]);
  }
  *reinterpret_cast<uint2*>(out + row_at + ch) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// The tokens first, first + stride, .. below `tokens` of a cluster's tile, by one warp.  `parts` CTAs of the cluster (every step-th from
// `from` on, which may differ from lane to lane; `remote`: there are others than this one) hold sums of a token, four channels of each of
// HALVES for this lane, at the shared memory address base + pitch * token + apart * half of their own.  They are added in the order of the
// CTAs and given to store(token, v).  Several tokens' sums are on their way at a time: a read of another CTA's shared memory takes a few
// hundred cycles.
template <int HALVES, int MOST, typename Store>
__device__ __forceinline__ void join_tokens(int first, int stride, int tokens, int parts, int from, int step, bool remote, uint32_t base,
                                            uint32_t pitch, uint32_t apart, Store store) {
  auto go = [&](auto parts_c) {
    constexpr int P = decltype(parts_c)::value, U = 8 / HALVES / P > 0 ? 8 / HALVES / P : 1;
    for (int t0 = first; t0 < tokens; t0 += stride * U) {
      float4 part[U][P][HALVES];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = min(t0 + stride * u, tokens - 1);
#pragma unroll
        for (int s = 0; s < P; ++s) {
          if (s < parts) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              const uint32_t at = base + pitch * t + apart * h;
              part[u][s][h] = ptx::ld_cluster_f4(remote ? ptx::mapa(at, from + step * s) : at);
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t0 + stride * u < tokens) {
          float v[HALVES][4];
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            v[h][0] = part[u][0][h].x;
            v[h][1] = part[u][0][h].y;
            v[h][2] = part[u][0][h].z;
            v[h][3] = part[u][0][h].w;
#pragma unroll
            for (int s = 1; s < P; ++s) {
              if (s < parts) {
                v[h][0] += part[u][s][h].x;
                v[h][1] += part[u][s][h].y;
                v[h][2] += part[u][s][h].z;
                v[h][3] += part[u][s][h].w;
              }
            }
          }
          store(t0 + stride * u, v);
        }
      }
    }
  };
  if (parts == 1) go(std::integral_constant<int, 1>{});
  else if (parts == 2) go(std::integral_constant<int, 2>{});
  else if (parts <= 4) go(std::integral_constant<int, 4>{});
  else if constexpr (MOST > 4) go(std::integral_constant<int, 8>{});
}

// A warp has 128 gate and 128 up sums of a token, four of each per lane: activation, the group's scale, e4m3.
__device__ __forceinline__ void store_gated(const float (&v)[2][4], int activation, uint8_t* out, float* scale) {
  const int lane = threadIdx.x & 31;
  float h[4], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = act_mul_fast(v[0][i], v[1][i], activation);
    amax = fmaxf(amax, fabsf(h[i]));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  const float s = group_scale(amax);
  *reinterpret_cast<uint32_t*>(out + 4 * lane) = quant4(h, s, __frcp_rn(s), amax <= 3.0e38f);
  if (lane == 0) *scale = s;
}
#endif

}  // namespace fmoe
