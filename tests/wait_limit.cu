// A kernel whose waits never complete, for the test of what a wait that runs
// out leaves behind: warp 0 waits on a barrier that nothing arrives at, with a
// limit of its own; warp 1 on another, with the default one, and is to follow
// as soon as warp 0 has given up.  out: whether each wait completed, and
// whether one on a barrier that has completed did.
#include <cuda_runtime.h>

#include "sm100.cuh"

using namespace tv::sm100;

__global__ void wait_limit_kernel(int* status, int* out, long long limit) {
  __shared__ uint64_t bars[3];
  __shared__ int abort_word;
  volatile int* abort = &abort_word;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();
    abort_word = 0;
    mbar_arrive(&bars[2]);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    out[2] = mbar_wait_suspend(&bars[2], 0, abort, limit);
    out[0] = mbar_wait_suspend(&bars[0], 0, abort, limit);
    if (!out[0]) give_up(abort, status, 3);
  } else if (threadIdx.x == 32) {
    out[1] = mbar_wait_suspend(&bars[1], 0, abort);
    if (!out[1]) give_up(abort, status, 4);
  }
}

extern "C" int run_wait_limit(int* status, int* out, long long limit, void* stream) {
  wait_limit_kernel<<<1, 64, 0, static_cast<cudaStream_t>(stream)>>>(status, out, limit);
  return cudaGetLastError();
}
