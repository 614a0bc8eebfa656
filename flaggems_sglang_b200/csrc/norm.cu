// Residual addition, root-mean-square norm and quantisation to e4m3 in one pass over the rows:
//     h = round(x + r);  y = h / sqrt(mean(h^2) + eps) * w;  q = e4m3(y / s), s = max(amax(y), 1e-10) / 448 per 128 channels
//     (or one s per row), norm = round(y)
// (quotients: rows.cuh)
// A CTA owns a row at a time and keeps it in registers between the sum of squares and the outputs, so every byte is read and
// written once: HBM bounds it from some ten MB on (beside the issue slots, where a row has neither residual nor norm to move), the
// launch and the dependent reductions below that: one row of 7168 takes 3 us.  Rows of which only the quantised norm is wanted run at 0.4
// to 0.6 of the copy rate (8192 rows of 7168 bf16 58 us): 26 instructions per value, 70 % of the issue slots.  Two values per instruction
// (f32x2), four vectors per thread instead of two, or no bounds predicates change that by 5 % at most, and cost rows with a residual as much.
#include <algorithm>
#include <type_traits>

#include "ptx_sm100.cuh"
#include "rows.cuh"

namespace fmoe {

// This translation unit's status word; read by status_word_norm().
__device__ int g_device_status_norm = 0;

namespace {

constexpr int kMaxStages = 4;
constexpr int kStreamBytes = 220 * 1024;  // shared memory of an SM for the rows on their way
__device__ __forceinline__ void report(int code) { atomicCAS(&g_device_status_norm, 0, code); }

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
  float eps, inv_K;
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
// False, to every thread, if any thread's `fine` is.
template <bool MAX>
__device__ __forceinline__ bool cta_reduce(float& v, float* buf, bool fine) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) buf[threadIdx.x >> 5] = v;
  fine = __syncthreads_and(fine);
  v = lane < warps ? buf[lane] : 0.f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  return fine;
}

// The rest of a row whose sums h are in registers: sum of squares, norm, scales, e4m3.  `fine` (of this thread) is false where
// its loads did not arrive; false is returned to every thread then, and nothing of the row has been written here.
template <typename T, int VECS, bool PER_TOKEN>
__device__ __forceinline__ bool finish_row(const NormParams& p, int64_t row, float (&h)[VECS][8], float (*buf)[32], bool fine) {
  const int vecs = p.K / 8;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
  }
  if (!cta_reduce<false>(sum, buf[0], fine)) return false;
  const float rstd = rsqrtf(fmaf(sum, p.inv_K, p.eps));
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
    cta_reduce<true>(amax_row, buf[1], true);
    s_row = fmaxf(scale_448(amax_row), 1.0f / (448.0f * 512.0f));
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
      s = scale_448(fmaxf(amax, 1e-10f));
    }
    if (c < vecs) {
      *reinterpret_cast<uint2*>(p.q + row * p.K + 8 * c) = quant8_corrected(h[i], s, amax <= 3.0e38f);
      if (!PER_TOKEN && c % 16 == 0) p.scale[row * (p.K / 128) + c / 16] = s;
    }
  }
  if constexpr (!PER_TOKEN) __syncthreads();  // the warps' sums have been read by everyone (PER_TOKEN: cta_reduce's barrier)
  return true;
}

// h = x, or round(x + r) which is stored
template <typename T, int VECS>
__device__ __forceinline__ void add_residual(const NormParams& p, T* res, float (&h)[VECS][8], const float (&r)[VECS][8]) {
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (8 * c < p.K) {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = to_f32(from_f32<T>(h[i][j] + r[i][j]));
      store8(res + 8 * c, h[i]);
    }
  }
}

// A CTA per row, loads straight into registers.  MAX_THREADS 448: three CTAs of so many threads on an SM (40 registers).
template <typename T, int VECS, bool PER_TOKEN, bool RESIDUAL, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS, MAX_THREADS == 448 ? 3 : 1)
rms_norm_quant_kernel(const NormParams p) {
  pdl_entry_late();
  __shared__ float buf[2][32];
  const int vecs = p.K / 8;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    T* res = RESIDUAL ? reinterpret_cast<T*>(p.residual) + row * p.residual_stride : nullptr;
    float h[VECS][8], r[VECS][8];
    // every load of the row is on its way before the first sum is stored
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
      if (c < vecs) {
        load8(x + 8 * c, h[i]);
        if constexpr (RESIDUAL) load8(res + 8 * c, r[i]);
      }
    }
    if constexpr (RESIDUAL) add_residual<T, VECS>(p, res, h, r);
    finish_row<T, VECS, PER_TOKEN>(p, row, h, buf, true);
  }
}

// Long bf16 rows: persistent CTAs whose rows arrive in a ring of shared memory (one bulk copy per row and tensor), so that the next
// rows' bytes are on their way while this one is reduced.  With residual and norm 8192 rows of 7168 take 98 us with loads into registers (two
// CTAs of 448 threads fit an SM), 90 us here, 5.9 TB/s; of 6144, where three CTAs fit, 74 and 79, of 2944 37 and 42.
// MAX_THREADS 512, 768: three and two CTAs of so many threads on an SM (40 registers); 1024: one (52), or two of up to 576.
template <bool PER_TOKEN, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS, 1536 / MAX_THREADS)
rms_norm_quant_stream_kernel(const NormParams p, int stages) {
  using T = __nv_bfloat16;
  constexpr int VECS = 2;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float buf[2][32];
  __shared__ uint64_t full[kMaxStages];
  const int vecs = p.K / 8, row_bytes = p.K * (int)sizeof(T), stage_bytes = row_bytes * (p.residual ? 2 : 1);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) ptx::mbar_init(&full[s], 1);
    ptx::fence_barrier_init();
  }
  __syncthreads();
  pdl_entry_late();
  auto fetch = [&](int64_t row, int s) {
    ptx::mbar_arrive_expect_tx(&full[s], stage_bytes);
    ptx::bulk_load(ptx::smem_u32(ring + s * stage_bytes), reinterpret_cast<const T*>(p.x) + row * p.x_stride, row_bytes, ptx::smem_u32(&full[s]));
    if (p.residual)
      ptx::bulk_load(ptx::smem_u32(ring + s * stage_bytes + row_bytes), reinterpret_cast<const T*>(p.residual) + row * p.residual_stride, row_bytes,
                     ptx::smem_u32(&full[s]));
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s)
      if (blockIdx.x + (int64_t)s * gridDim.x < p.rows) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  }
  int stage = 0;
  uint32_t phase = 0;
  int64_t next = blockIdx.x + (int64_t)stages * gridDim.x;
  bool alive = true;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, next += gridDim.x) {
    T* res = p.residual ? reinterpret_cast<T*>(p.residual) + row * p.residual_stride : nullptr;
    const T* x = reinterpret_cast<const T*>(ring + stage * stage_bytes);
    float h[VECS][8];
    bool fine = ptx::mbar_wait(&full[stage], phase);
    // all threads agree before the first store, and again in the sum of squares, which all of them have read the stage for
    if (res && !__syncthreads_and(fine)) {
      alive = false;
      break;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
      if (c < vecs) {
        load8(x + 8 * c, h[i]);
        if (res) {
          float r[8];
          load8(reinterpret_cast<const T*>(ring + stage * stage_bytes + row_bytes) + 8 * c, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[i][j] = to_f32(from_f32<T>(h[i][j] + r[j]));
          store8(res + 8 * c, h[i]);
        }
      }
    }
    if (!finish_row<T, VECS, PER_TOKEN>(p, row, h, buf, fine)) {
      alive = false;
      break;
    }
    if (threadIdx.x == 0 && next < p.rows) fetch(next, stage);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (!alive && threadIdx.x == 0) {
    report(0x3100);
    for (int s = 0; s < stages; ++s) ptx::mbar_wait(&full[s], s < stage ? phase ^ 1 : phase);  // copies still on their way
  }
}

// Whether rows of K elements from a and from b have memory in common.  Interleaved rows of the same stride (halves of one buffer's) need
// not, though the ranges from first to last do.
bool rows_meet(const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t rows, int64_t K, int64_t size) {
  const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));  // bytes
  const int64_t a_len = ((rows - 1) * a_stride + K) * size, b_len = ((rows - 1) * b_stride + K) * size;
  if (apart >= a_len || -apart >= b_len) return false;
  if (rows == 1 || a_stride != b_stride) return true;
  const int64_t pitch = a_stride * size, in_row = ((apart % pitch) + pitch) % pitch;
  return in_row < K * size || in_row > pitch - K * size;
}

}  // namespace

int status_word_norm(int* out, bool clear);

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
  FMOE_REQUIRE(!residual || (residual == x && residual_stride == x_stride) ||
                   !rows_meet(x, x_stride, residual, residual_stride, rows, K, dtype == FMOE_BF16 ? 2 : 4),
               "rms_norm_quant: residual shares memory with other rows of x");
  NormParams p{x, residual, weight, (uint8_t*)q, scale, norm, x_stride, residual_stride, rows, (int)K, weight_dtype == FMOE_F32, eps, 1.0f / (float)K};
  const int vecs = (int)(K / 8);
  const auto st = (cudaStream_t)stream;
  auto threads = [&](int v) { return (unsigned)(ceil_div(ceil_div(vecs, v), 32) * 32); };
  auto each_type = [&](auto go) {  // go(type, per_token)
    if (dtype == FMOE_BF16) per_token ? go((__nv_bfloat16*)nullptr, std::true_type{}) : go((__nv_bfloat16*)nullptr, std::false_type{});
    else per_token ? go((float*)nullptr, std::true_type{}) : go((float*)nullptr, std::false_type{});
  };
  // Many rows (us of 8192 without residual; in registers, there with three CTAs of up to 448 threads, by the ring): bf16 4096 channels 34.5,
  // 31.2, 37.1, 7168 67.8, 58.3, 61.6; fp32 4096 36.0, 37.4, 7168 76.2, 68.8.  With residual that many registers do not do.
  const bool many = rows > 296, three = many && !residual && threads(2) <= 448 && (dtype == FMOE_BF16 || threads(2) > 256);
  if (dtype == FMOE_BF16 && many && !three && (!residual || threads(2) > 384)) {
    const int stage_bytes = (int)K * 2 * (residual ? 2 : 1);
    // Above 576 threads two CTAs fit with 40 registers, not with 52: 8192 rows of 9728 with residual 118 us and 134, of 12288 150 and 153,
    // without 82 and 95, 97 and 105; of 8704 (544 threads, two fit either way) 108 and 106, 77 and 72.  With a scale per row 40 registers
    // spill (12288 with residual 161 and 153, 9728 132 and 133, without 88 and 94): the larger kernel, half of whose CTAs wait.
    const int ctas = std::min(std::max(1, 1536 / (int)threads(2)), (kStreamBytes - 2048) / (2 * stage_bytes + 1024));  // at least 1: K <= 16384
    const int stages = std::min(kMaxStages, (kStreamBytes / ctas - 1024) / stage_bytes);
    cudaError_t attr_err = cudaSuccess;
    auto go = [&](auto token) {
      constexpr bool PER_TOKEN = decltype(token)::value;
      auto kernel = rms_norm_quant_stream_kernel<PER_TOKEN, 512>;
      auto wide = rms_norm_quant_stream_kernel<PER_TOKEN, 1024>;
      auto middle = rms_norm_quant_stream_kernel<false, 768>;
      static PerDeviceOnce once_attr;
      attr_err = per_device_once(once_attr, [&] {
        cudaError_t e = cudaSuccess;
        for (auto k : {kernel, middle, wide})
          if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamBytes);
        return e;
      });
      if (attr_err != cudaSuccess) return;
      const unsigned grid = (unsigned)std::min<int64_t>(rows, (int64_t)148 * ctas);
      const bool two = !PER_TOKEN && threads(2) > 576 && threads(2) <= 768;
      launch_pdl(two ? middle : (threads(2) > 512 ? wide : kernel), dim3(grid), dim3(threads(2)), (size_t)stages * stage_bytes, st, p, stages);
    };
    if (per_token) go(std::true_type{});
    else go(std::false_type{});
    if (attr_err != cudaSuccess) return fail(FMOE_ERR_CUDA, "set-up of the norm kernel failed: %s", cudaGetErrorString(attr_err));
    return launch_status("rms_norm_quant_stream_kernel");
  }
  each_type([&](auto* type, auto token) {
    using E = std::remove_pointer_t<decltype(type)>;
    auto with = [&](auto v) {
      constexpr int VV = decltype(v)::value;
      constexpr bool PER_TOKEN = decltype(token)::value;
      auto kernel = residual ? rms_norm_quant_kernel<E, VV, PER_TOKEN, true, 1024> : rms_norm_quant_kernel<E, VV, PER_TOKEN, false, 1024>;
      if constexpr (VV == 2)
        if (three) kernel = rms_norm_quant_kernel<E, 2, PER_TOKEN, false, 448>;
      launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(rows, 148 * 32)), dim3(threads(VV)), 0, st, p);
    };
    if (vecs <= 1024 && !many) with(std::integral_constant<int, 1>{});
    else with(std::integral_constant<int, 2>{});
  });
  return launch_status("rms_norm_quant_kernel");
}

int fmoe::status_word_norm(int* out, bool clear) {
  int zero = 0;
  FMOE_CUDA_OK(cudaMemcpyFromSymbol(out, fmoe::g_device_status_norm, sizeof(int)));
  if (clear && *out != 0) FMOE_CUDA_OK(cudaMemcpyToSymbol(fmoe::g_device_status_norm, &zero, sizeof(int)));
  return FMOE_OK;
}
