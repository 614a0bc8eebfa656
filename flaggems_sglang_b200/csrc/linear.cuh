// Internal interface of the dense e4m3 products (linear.cu).
#pragma once
#include "gemm.cuh"

namespace fmoe {

// One product of e4m3 rows with e4m3 weights.  gated: `w` has 2n rows (gate rows, then up rows), the output is the quantised
// activation [T, n]; otherwise n rows, the output is bf16 [T, n].
struct LinearParams {
  int64_t T = 0, n = 0, k = 0;
  const void* x = nullptr;         // [T, k] e4m3
  const float* x_scale = nullptr;  // [T, k/128]
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
int run_linear(const LinearParams& p, bool gated, cudaStream_t st);

}  // namespace fmoe
