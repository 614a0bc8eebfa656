// A kernel that lets its successor on the stream start at once, and runs on for a number of clocks.
#include <cuda_runtime.h>

static __global__ void early_trigger_kernel(long long clocks) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long t0 = clock64();
  for (int i = 0; i < (1 << 22) && clock64() - t0 < clocks; ++i) __nanosleep(1000);
}

extern "C" int early_trigger(long long clocks, void* stream) {
  early_trigger_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(clocks);
  return (int)cudaGetLastError();
}
