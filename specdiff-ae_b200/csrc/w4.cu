// Rows times 4-bit weights with group scales:
//
//   y[t, n] = xs[t] * sum_k x[t, k] * (u[n, k] - 8) * s[n, k / group]
//
// One warp per weight row and block of tokens: a lane takes every 32nd word of
// eight weights, sums its products in fp32 and scales each word's sum.
#include <cuda_fp8.h>

#include "common.cuh"

namespace tv {
namespace {

constexpr int kTokens = 4;       // tokens per warp

struct W4Params {
  const void* x;
  int64_t x_sm;
  const float* x_scale;
  const uint32_t* q;
  int64_t q_sn;
  const void* s;
  int64_t s_sn;
  void* out;
  int64_t o_sm;
  int rows, n, k, group;
};

template <typename X> __device__ __forceinline__ float x_float(X v) { return Elem<X>::to_f(v); }
template <> __device__ __forceinline__ float x_float<__nv_fp8_e4m3>(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

template <typename X, typename T>
__global__ void __launch_bounds__(256) w4_kernel(const W4Params a) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t0 = blockIdx.y * kTokens;
  if (n >= a.n) return;
  const uint32_t* q = a.q + (int64_t)n * a.q_sn;
  const T* s = static_cast<const T*>(a.s) + (int64_t)n * a.s_sn;
  float acc[kTokens] = {};
  for (int c = lane; c < a.k / 8; c += 32) {
    const uint32_t w = q[c];
    const float sc = Elem<T>::to_f(s[c * 8 / a.group]);
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (t0 + i >= a.rows) break;
      const X* x = static_cast<const X*>(a.x) + (int64_t)(t0 + i) * a.x_sm + c * 8;
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d = fmaf(x_float<X>(x[2 * j]), (float)((int)((w >> (4 * j)) & 15) - 8), d);
        d = fmaf(x_float<X>(x[2 * j + 1]), (float)((int)((w >> (4 * j + 16)) & 15) - 8), d);
      }
      acc[i] = fmaf(d, sc, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (lane == 0 && t0 + i < a.rows)
      static_cast<T*>(a.out)[(int64_t)(t0 + i) * a.o_sm + n] =
          Elem<T>::from_f(acc[i] * (a.x_scale ? a.x_scale[t0 + i] : 1.f));
  }
}

template <typename X, typename T>
int launch_w4(const W4Params& p, cudaStream_t st) {
  w4_kernel<X, T><<<dim3((p.n + 7) / 8, (p.rows + kTokens - 1) / kTokens), 256, 0, st>>>(p);
  return check_launch();
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" {

int tv_w4_workspace_size(const tv_w4_args* a, size_t* bytes) {
  if (!a || !bytes) return TV_ERR_NULL;
  *bytes = 0;
  return TV_OK;
}

int tv_w4_linear(const tv_w4_args* a, void* stream) {
  if (!a) return TV_ERR_NULL;
  if (a->rows < 0 || a->n < 1 || a->group < 32 || a->group % 32 != 0 || a->k < a->group || a->k % a->group != 0)
    return TV_ERR_SHAPE;
  if (a->out_dtype != TV_BF16 && a->out_dtype != TV_F16) return TV_ERR_DTYPE;
  if (a->x_dtype != a->out_dtype && a->x_dtype != TV_E4M3) return TV_ERR_DTYPE;
  if (a->rows == 0) return TV_OK;
  if (!a->x || !a->qweight || !a->scales || !a->out || (a->x_dtype == TV_E4M3 && !a->x_scale)) return TV_ERR_NULL;
  if (!aligned16(a->qweight) || a->q_sn % 4 != 0) return TV_ERR_ALIGN;
  if (a->rows > 65535 * kTokens) return TV_ERR_UNSUPPORTED;
  const W4Params p{a->x, a->x_sm, a->x_scale, static_cast<const uint32_t*>(a->qweight), a->q_sn, a->scales, a->s_sn,
                   a->out, a->o_sm, a->rows, a->n, a->k, a->group};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->out_dtype == TV_BF16)
    return a->x_dtype == TV_E4M3 ? launch_w4<__nv_fp8_e4m3, __nv_bfloat16>(p, st)
                                 : launch_w4<__nv_bfloat16, __nv_bfloat16>(p, st);
  return a->x_dtype == TV_E4M3 ? launch_w4<__nv_fp8_e4m3, __half>(p, st) : launch_w4<__half, __half>(p, st);
}

}  // extern "C"
