// Residual addition, root-mean-square norm and quantisation to e4m3 in one pass over the rows:
//     h = round(x + r);  y = h / sqrt(mean(h^2) + eps) * w;  q = e4m3(y / s), s = max(amax(y), 1e-10) / 448 per 128 channels
//     (or one s per row), norm = round(y)
// A CTA owns a row at a time and keeps it in registers between the sum of squares and the outputs, so every byte is read and
// written once: HBM bounds it from a few MB on, the launch and two dependent reductions below that.
#include <algorithm>

#include "rows.cuh"

namespace fmoe {
namespace {

struct NormParams {
  const void* x;
  void* residual;
  const void* weight;
  uint8_t* q;
  float* scale;
  void* norm;
  int64_t x_stride, residual_stride, rows;
  int K;
  int weight_f32;
  float eps;
};

// eight consecutive values
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __low2float(h[i]);
    v[2 * i + 1] = __high2float(h[i]);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Reduction over the CTA's warps, the same value in every thread.  `buf` holds a value per warp; two calls in a row use two.
template <bool MAX>
__device__ __forceinline__ float cta_reduce(float v, float* buf) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? buf[lane] : 0.f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  return v;
}

template <typename T, int VECS, bool PER_TOKEN>
__global__ void __launch_bounds__(1024)
rms_norm_quant_kernel(const NormParams p) {
  pdl_entry_late();
  __shared__ float buf[2][32];
  const int vecs = p.K / 8;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    T* res = p.residual ? reinterpret_cast<T*>(p.residual) + row * p.residual_stride : nullptr;
    float h[VECS][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
      if (c < vecs) {
        load8(x + 8 * c, h[i]);
        if (res) {
          float r[8];
          load8(res + 8 * c, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[i][j] = to_f32(from_f32<T>(h[i][j] + r[j]));
          store8(res + 8 * c, h[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    }
    sum = cta_reduce<false>(sum, buf[0]);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sum, (float)p.K) + p.eps));
    float amax_row = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < vecs) {
        float w[8];
        if (p.weight_f32) load8(reinterpret_cast<const float*>(p.weight) + 8 * c, w);
        else load8(reinterpret_cast<const __nv_bfloat16*>(p.weight) + 8 * c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[i][j] = h[i][j] * rstd * w[j];
          if (PER_TOKEN) amax_row = fmaxf(amax_row, fabsf(h[i][j]));
        }
        if (p.norm) store8(reinterpret_cast<T*>(p.norm) + row * p.K + 8 * c, h[i]);
      }
    }
    float s_row = 0.f;
    if constexpr (PER_TOKEN) {
      amax_row = cta_reduce<true>(amax_row, buf[1]);
      s_row = fmaxf(__fdiv_rn(amax_row, 448.0f), 1.0f / (448.0f * 512.0f));
      if (threadIdx.x == 0) p.scale[row] = s_row;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      float amax = amax_row, s = s_row;
      if constexpr (!PER_TOKEN) {  // a group is the vectors of 16 neighbouring lanes: K is a multiple of 128
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(h[i][j]));
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        s = group_scale(amax);
      }
      if (c < vecs) {
        *reinterpret_cast<uint2*>(p.q + row * p.K + 8 * c) = quant8(h[i], s, __frcp_rn(s), amax <= 3.0e38f);
        if (!PER_TOKEN && c % 16 == 0) p.scale[row * (p.K / 128) + c / 16] = s;
      }
    }
    if constexpr (!PER_TOKEN) __syncthreads();  // the sums of this row have been read by everyone (PER_TOKEN: cta_reduce's barrier)
  }
}

}  // namespace
}  // namespace fmoe

extern "C" int fmoe_rms_norm_quant(const void* x, int64_t x_stride, void* residual, int64_t residual_stride, int dtype, const void* weight,
                                   int weight_dtype, int64_t rows, int64_t K, float eps, int per_token, void* q, float* scale, void* norm,
                                   void* stream) {
  using namespace fmoe;
  FMOE_REQUIRE(dtype == FMOE_BF16 || dtype == FMOE_F32, "rms_norm_quant: x must be bf16 or f32");
  FMOE_REQUIRE(weight_dtype == FMOE_BF16 || weight_dtype == FMOE_F32, "rms_norm_quant: weight must be bf16 or f32");
  FMOE_REQUIRE(K > 0 && K <= 16384 && K % (per_token ? 8 : 128) == 0, "rms_norm_quant: K must be a multiple of %d up to 16384 (got %lld)",
               per_token ? 8 : 128, (long long)K);
  FMOE_REQUIRE(rows >= 0 && rows < (1ll << 31), "rms_norm_quant: bad number of rows %lld", (long long)rows);
  FMOE_REQUIRE(eps >= 0.f, "rms_norm_quant: eps must be >= 0");
  const int per16 = dtype == FMOE_BF16 ? 8 : 4;
  FMOE_REQUIRE(x_stride >= K && x_stride % per16 == 0 && (!residual || (residual_stride >= K && residual_stride % per16 == 0)),
               "rms_norm_quant: row strides must be at least K and multiples of 16 bytes");
  if (rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x && weight && q && scale, "rms_norm_quant: null pointer");
  FMOE_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(norm) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 &&
                   (reinterpret_cast<uintptr_t>(scale) & 3u) == 0,
               "rms_norm_quant: misaligned pointer");
  NormParams p{x, residual, weight, (uint8_t*)q, scale, norm, x_stride, residual_stride, rows, (int)K, weight_dtype == FMOE_F32, eps};
  const int vecs = (int)(K / 8);
  auto go = [&](auto vecs_c) {
    constexpr int V = decltype(vecs_c)::value;
    const unsigned threads = (unsigned)(ceil_div(ceil_div(vecs, V), 32) * 32);
    const unsigned grid = (unsigned)std::min<int64_t>(rows, 148 * 32);
    auto with = [&](auto kernel) { launch_pdl(kernel, dim3(grid), dim3(threads), 0, (cudaStream_t)stream, p); };
    if (dtype == FMOE_BF16) per_token ? with(rms_norm_quant_kernel<__nv_bfloat16, V, true>) : with(rms_norm_quant_kernel<__nv_bfloat16, V, false>);
    else per_token ? with(rms_norm_quant_kernel<float, V, true>) : with(rms_norm_quant_kernel<float, V, false>);
  };
  if (vecs <= 1024) go(std::integral_constant<int, 1>{});
  else go(std::integral_constant<int, 2>{});
  return launch_status("rms_norm_quant_kernel");
}
