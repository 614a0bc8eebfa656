// Internal interface of the row kernels (rows.cu).
#pragma once
#include "common.cuh"

namespace fmoe {

// The layer's passes, by slot: slot_pos [T * k] is every slot's position in the sorted order (-1: none), as run_align
// writes it; padding positions are neither read nor written.
// token rows -> the positions of their k slots
int run_scatter_rows(const void* x, int elem_bytes, int64_t T, int k, int64_t K, const int32_t* slot_pos, void* out, cudaStream_t st);
// bf16 token rows -> e4m3 at the positions of their k slots; scales by token: [T, K/128], or [T] with per_row
int run_quant_scatter(const void* x, int64_t T, int k, int64_t K, const int32_t* slot_pos, bool per_row, void* q, float* scale,
                      cudaStream_t st);
// sorted bf16 rows -> e4m3 with one scale per row, in the same positions, scales by position
int run_quant_rows(const void* x, int64_t numel, int64_t K, const int32_t* slot_pos, void* q, float* scale, cudaStream_t st);
// sorted f32 rows -> e4m3 with a scale per 128 channels, likewise
int run_quant_slots(const float* x, int64_t numel, int64_t K, const int32_t* slot_pos, void* q, float* scale, cudaStream_t st);
// the same from max_rows f32 rows per expert to the experts' positions, only the experts with up to max_rows rows (table: pair.cuh): CTAs per expert, so that the other experts cost nothing
// (DeepSeek-V3, 4096 tokens, a third of the experts: 21 us against 105 us of looking at every slot)
int run_quant_experts(const float* x, int64_t numel, int64_t K, int num_experts, const int32_t* table, int max_rows, void* q,
                      float* scale, cudaStream_t st);

// bf16 rows -> e4m3 with a scale per 128 channels; the next kernel starts only after this one's own wait
int run_quant_tokens(const void* x, int64_t T, int64_t K, void* q, float* scale, cudaStream_t st);

#if defined(__CUDACC__)
// Scale of a group of 128 channels with this largest magnitude.
__device__ __forceinline__ float group_scale(float amax) { return __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f); }

// Eight values divided by the scale s (r = 1/s rounded) and rounded to e4m3; `finite`: none of the group is infinite.
__device__ __forceinline__ uint2 quant8(const float (&v)[8], float s, float r, bool finite) {
  uint32_t lo = 0, hi = 0;
  if (finite) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = div_by_shared(v[i], s, r);
    // two values per conversion instruction (low byte = first value)
    auto pair = [](float a, float b) {
      return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    };
    lo = pair(q[0], q[1]) | (pair(q[2], q[3]) << 16);
    hi = pair(q[4], q[5]) | (pair(q[6], q[7]) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo |= (uint32_t)f32_to_e4m3_bits(__fdiv_rn(v[i], s)) << (8 * i);
      hi |= (uint32_t)f32_to_e4m3_bits(__fdiv_rn(v[4 + i], s)) << (8 * i);
    }
  }
  return make_uint2(lo, hi);
}

// Division costs most of the instructions of a quantiser that is written with __fdiv_rn (the norm: 42 per value in all, issue slots 74 %
// busy, 93 us for 8192 rows of 7168).  Here a quotient is a product with the reciprocal and one correction by its exact remainder
// (Markstein's, of which div_by_shared does two).  Before the last rounding it is off by what the reciprocal and the first product are
// off by, times what the reciprocal is off by: by __fdividef (2 ulp, 2^-22) 1.25 * 2^-44 of itself, 2^-20 of a unit in the last
// place or so, by a correctly rounded reciprocal 2^-23.  It differs from the correctly rounded quotient at most where that lies as close to
// the middle of two floats: by the constant 448 for no significand, so that scales are the same bits, nor are any e4m3 values of bf16
// rows (tests compare all 2^23, and all pairs of significands 24 exponents apart).  (The norm's fp32 values have no such proof: there
// an e4m3 value may differ where y / s lies that close to a tie, which the rounding of y moves by more.)
__device__ __forceinline__ float corrected_quotient(float v, float d, float r) {
  const float q = v * r;
  return fmaf(fmaf(-q, d, v), r, q);
}
// max / 448
__device__ __forceinline__ float scale_448(float amax) {
  return amax <= 3.0e38f ? corrected_quotient(amax, 448.0f, 1.0f / 448.0f) : __fdiv_rn(amax, 448.0f);
}
// eight values over s -> e4m3; `finite`: none of the group is infinite
__device__ __forceinline__ uint2 quant8_corrected(const float (&v)[8], float s, bool finite) {
  if (!finite) return quant8(v, s, 0.f, false);
  const float r = __fdividef(1.0f, s);
  uint32_t half[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    half[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(corrected_quotient(v[2 * i], s, r), corrected_quotient(v[2 * i + 1], s, r)),
                                                 __NV_SATFINITE, __NV_E4M3);
  return make_uint2(half[0] | half[1] << 16, half[2] | half[3] << 16);
}

// U groups of 128 bf16 channels, 16 channels of each of eight neighbouring lanes: their e4m3 values, and the groups' scales in every lane.
// All 32 lanes call it.  Step by step over all groups, and infinities are mended behind: a branch between them would put the groups'
// dependent chains (shuffles, scale, reciprocal) one behind the other.
template <int U>
__device__ __forceinline__ void quant_groups(const uint4 (&raw)[U][2], uint4 (&packed)[U], float (&s)[U]) {
  float amax[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw[u]);
    __nv_bfloat162 m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __hmax2(__habs2(e[j]), __habs2(e[j + 4]));
    m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    amax[u] = fmaxf(fmaxf(__low2float(m[0]), __high2float(m[0])), 0.f);  // a group of nothing but NaN: as one of zeros
  }
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) {
#pragma unroll
    for (int u = 0; u < U; ++u) amax[u] = fmaxf(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], off));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) s[u] = corrected_quotient(fmaxf(amax[u], 1e-10f), 448.0f, 1.0f / 448.0f);
  auto value8 = [&](const uint4& part, float (&v)[8]) {
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&part);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __low2float(e[j]);
      v[2 * j + 1] = __high2float(e[j]);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[2][8];
    value8(raw[u][0], v[0]);
    value8(raw[u][1], v[1]);
    const uint2 lo = quant8_corrected(v[0], s[u], true), hi = quant8_corrected(v[1], s[u], true);
    packed[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!(amax[u] <= 3.0e38f)) {
      s[u] = scale_448(amax[u]);
      float v[2][8];
      value8(raw[u][0], v[0]);
      value8(raw[u][1], v[1]);
      const uint2 lo = quant8(v[0], s[u], 0.f, false), hi = quant8(v[1], s[u], 0.f, false);
      packed[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
}

// Four values as quant8.
__device__ __forceinline__ uint32_t quant4(const float (&v)[4], float s, float r, bool finite) {
  uint32_t w = 0;
  if (finite) {
    auto pair = [](float a, float b) {
      return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    };
    w = pair(div_by_shared(v[0], s, r), div_by_shared(v[1], s, r)) | (pair(div_by_shared(v[2], s, r), div_by_shared(v[3], s, r)) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)f32_to_e4m3_bits(__fdiv_rn(v[i], s)) << (8 * i);
  }
  return w;
}
#endif

}  // namespace fmoe
