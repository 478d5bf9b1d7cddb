// Row-wise elementwise work of the target's decoder layers around the verify
// path, one launch each: LlamaRMSNorm (runtime/llama_target_model.py:124-138)
// and the SwiGLU gate act_fn(gate) * up of LlamaMLP (:506-538), with the
// reference's roundings (fp32 statistics, the normalised row rounded to the
// element type before the weight multiply; silu rounded before the product).
//
// One CTA per row for the norm (the row's sum of squares is a block
// reduction); the gate is a flat grid over 8-element chunks.  Rows are read
// as 16-byte vectors: columns a multiple of 8, rows 16-byte aligned.
//
// tv_add_rms_norm takes the residual's addition in front of the norm into the
// same pass and can hand the row on in 8 bits with its scale.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "specverify.h"

namespace tv {
namespace {

constexpr int kNormThreads = 256;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = Elem<T>::to_f(e[k]);
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = Elem<T>::pack2(f[2 * k], f[2 * k + 1]);
  return u;
}

template <typename T>
__device__ __forceinline__ float round_to(float x) {
  return Elem<T>::to_f(Elem<T>::from_f(x));
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) rms_norm_kernel(const T* __restrict__ x, int64_t xs,
                                                                const T* __restrict__ w, T* __restrict__ y,
                                                                int64_t ys, int cols, float eps) {
  const T* xr = x + (int64_t)blockIdx.x * xs;
  T* yr = y + (int64_t)blockIdx.x * ys;
  float ss = 0.f;
  for (int c = threadIdx.x * 8; c < cols; c += kNormThreads * 8) {
    float f[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(xr + c), f);
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(f[k], f[k], ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  __shared__ float part[kNormThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) part[warp] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 32; ++i) tot += part[i];
  const float inv = rsqrtf(tot / (float)cols + eps);
  for (int c = threadIdx.x * 8; c < cols; c += kNormThreads * 8) {
    float f[8], g[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(xr + c), f);
    unpack8<T>(*reinterpret_cast<const uint4*>(w + c), g);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = round_to<T>(f[k] * inv) * g[k];
    *reinterpret_cast<uint4*>(yr + c) = pack8<T>(f);
  }
}

template <typename T>
__global__ void silu_mul_kernel(const T* __restrict__ g, const T* __restrict__ u, int64_t in_s, T* __restrict__ y,
                                int64_t out_s, int rows, int cols) {
  const int chunks = cols / 8;
  const int64_t n = (int64_t)rows * chunks;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    float a[8], b[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(g + r * in_s + c), a);
    unpack8<T>(*reinterpret_cast<const uint4*>(u + r * in_s + c), b);
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = round_to<T>(a[k] / (1.0f + expf(-a[k]))) * b[k];
    *reinterpret_cast<uint4*>(y + r * out_s + c) = pack8<T>(a);
  }
}

// ---- residual addition + RMSNorm ---------------------------------------------
//
//   h = T(x + r),  y = T(T(h * inv) * w),  inv = 1 / sqrt(mean(h^2) + eps)
// or, in 8 bits,
//   f = h * inv * w (fp32),  s = max|f| / 448,  y = e4m3(f / s).
//
// The norm is of the stored (rounded) stream h, so a later reader of h sees
// the row that was normalised; the 16-bit output rounds as tv_rms_norm does.
// One CTA per row.  A thread keeps its NC chunks of VEC elements of h in
// registers between the two passes, so every input is read once and every
// output written once: the kernel is bound by HBM for many rows and by
// latency (two or three block reductions) for few.
template <typename T, int VEC> struct Chunk;
template <typename T> struct Chunk<T, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ void get(float* f) const { unpack8<T>(v, f); }
  __device__ __forceinline__ void set(const float* f) { v = pack8<T>(f); }
};
template <typename T> struct Chunk<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float* f) const { f[0] = Elem<T>::to_f(v); }
  __device__ __forceinline__ void set(const float* f) { v = Elem<T>::from_f(f[0]); }
};

// Maximum that keeps a NaN of either side (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* f) {
  if constexpr (VEC == 8) {
    uint2 u;
    __nv_fp8x2_storage_t* e = reinterpret_cast<__nv_fp8x2_storage_t*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      e[k] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * k], f[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(p) = u;
  } else {
    *p = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
  }
}

struct AddNormArgs {
  const void* x;
  const void* r;
  const void* w;
  void* h;
  void* y;
  float* scale;
  int64_t xs, rs, hs, ys;
  int cols;
  float eps;
};

// NC chunks per thread stay in registers; WIDE rows (more than that) are read
// back from h, each thread its own chunks.
//
// SHIFT: rows that start off the 16-byte grid, x, r and h by the same offset
// (dense tensors with an odd number of columns).  The chunks begin at the
// row's first 16-byte boundary, the up to seven elements before and behind
// them go one to a thread, and what lies otherwise (the weight; y unless its
// offset is the same) is read or written element by element.
template <typename T, bool FP8, int VEC, int NC, bool WIDE, bool SHIFT>
__global__ void __launch_bounds__(512) add_rms_norm_kernel(const AddNormArgs a) {
  const T* x = static_cast<const T*>(a.x) + (int64_t)blockIdx.x * a.xs;
  const T* r = static_cast<const T*>(a.r) + (int64_t)blockIdx.x * a.rs;
  const T* w = static_cast<const T*>(a.w);
  T* h = static_cast<T*>(a.h) + (int64_t)blockIdx.x * a.hs;
  T* y = static_cast<T*>(a.y) + (int64_t)blockIdx.x * a.ys;
  uint8_t* y8 = static_cast<uint8_t*>(a.y) + (int64_t)blockIdx.x * a.ys;
  const int head = SHIFT ? min(a.cols, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T))) : 0;
  const int end = SHIFT ? head + (a.cols - head) / VEC * VEC : a.cols;      // of the chunks
  const int step = blockDim.x * VEC;
  const int first = head + threadIdx.x * VEC;
  // this thread's single element, if any
  const int single = !SHIFT ? -1
                     : (int)threadIdx.x < head ? (int)threadIdx.x
                     : end + (int)threadIdx.x - head < a.cols ? end + (int)threadIdx.x - head : -1;
  Chunk<T, VEC> keep[NC];
  Chunk<T, 1> one;
  float ss = 0.f;
  grid_next();
  grid_wait();
  // h = T(x + r), stored and squared
  auto join = [&](auto& u, const auto& v, int c) {
    constexpr int N = sizeof(u) / sizeof(T);
    float f[N], g[N];
    u.get(f);
    v.get(g);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] += g[k];
    u.set(f);
    u.store(h + c);
    u.get(f);
#pragma unroll
    for (int k = 0; k < N; ++k) ss = fmaf(f[k], f[k], ss);
  };
  if (!WIDE) {
    Chunk<T, VEC> cr[NC];
    Chunk<T, 1> cr1;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (first + i * step < end) {
        keep[i].load(x + first + i * step);
        cr[i].load(r + first + i * step);
      }
    if (SHIFT && single >= 0) {
      one.load(x + single);
      cr1.load(r + single);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (first + i * step < end) join(keep[i], cr[i], first + i * step);
    if (SHIFT && single >= 0) join(one, cr1, single);
  } else {
    for (int c = first; c < end; c += step) {
      Chunk<T, VEC> u, v;
      u.load(x + c);
      v.load(r + c);
      join(u, v, c);
    }
  }
  // What the thread holds of the row, chunk by chunk.
  auto each = [&](auto&& fn) {
    if (!WIDE) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (first + i * step < end) fn(keep[i], first + i * step);
      if (SHIFT && single >= 0) fn(one, single);
    } else {
      for (int c = first; c < end; c += step) {
        Chunk<T, VEC> u;
        u.load(h + c);
        fn(u, c);
      }
    }
  };
  auto weight = [&](int c, auto* g, auto n) {
    constexpr int N = decltype(n)::value;
    if constexpr (SHIFT && N > 1) {
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] = Elem<T>::to_f(w[c + k]);
    } else {
      Chunk<T, N> v;
      v.load(w + c);
      v.get(g);
    }
  };
  __shared__ float part[16];
  __shared__ float part_max[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) part[warp] = ss;
  __syncthreads();
  float tot = 0.f;
  for (int i = 0; i < warps; ++i) tot += part[i];
  const float inv = rsqrtf(tot / (float)a.cols + a.eps);

  if constexpr (!FP8) {
    const bool whole = !SHIFT || ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
    each([&](const auto& u, int c) {
      constexpr int N = sizeof(u) / sizeof(T);
      float f[N], g[N];
      weight(c, g, std::integral_constant<int, N>{});
      u.get(f);
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = round_to<T>(f[k] * inv) * g[k];
      if (whole) {
        Chunk<T, N> v;
        v.set(f);
        v.store(y + c);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) y[c + k] = Elem<T>::from_f(f[k]);
      }
    });
  } else {
    float mx = 0.f;
    each([&](const auto& u, int c) {
      constexpr int N = sizeof(u) / sizeof(T);
      float f[N], g[N];
      weight(c, g, std::integral_constant<int, N>{});
      u.get(f);
#pragma unroll
      for (int k = 0; k < N; ++k) mx = max_nan(mx, fabsf(f[k] * inv * g[k]));
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) part_max[warp] = mx;
    __syncthreads();
    mx = part_max[0];
    for (int i = 1; i < warps; ++i) mx = max_nan(mx, part_max[i]);
    const float s = mx * (1.0f / 448.0f);
    if (threadIdx.x == 0) a.scale[blockIdx.x] = s;
    // A row of zeros has scale 0 and stays zero.  The reciprocal of a scale
    // below 2^-100 is not safe to multiply with: divide there.
    const bool tiny = s < 7.8886091e-31f;
    const float is = 1.0f / s;
    each([&](const auto& u, int c) {
      constexpr int N = sizeof(u) / sizeof(T);
      float f[N], g[N];
      weight(c, g, std::integral_constant<int, N>{});
      u.get(f);
      if (tiny) {
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = s == 0.f ? 0.f : f[k] * inv * g[k] / s;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = f[k] * inv * g[k] * is;
      }
      if constexpr (SHIFT && N > 1) {
#pragma unroll
        for (int k = 0; k < N; ++k) store_e4m3<1>(y8 + c + k, f + k);
      } else {
        store_e4m3<N>(y8 + c, f);
      }
    });
  }
}

template <typename T, bool FP8, int VEC, int NC, bool WIDE, bool SHIFT>
int launch_add_norm(const AddNormArgs& a, int rows, int threads, cudaStream_t st) {
  return launch_early(add_rms_norm_kernel<T, FP8, VEC, NC, WIDE, SHIFT>, dim3((unsigned)rows), threads, 0, 0, st, a);
}

enum AddNormLayout { kRowsAligned, kRowsShifted, kRowsAny };

// Threads per row: as many as a row has chunks, at most 512; with enough rows
// to fill the GPU, a quarter of them with four chunks each (NCM: fewer warps
// meet at the reductions, and more rows are in flight per SM).  A row of more
// than 2048 chunks is read back from h.
template <typename T, bool FP8>
int pick_add_norm(const AddNormArgs& a, int rows, AddNormLayout layout, cudaStream_t st) {
  const int chunks = layout == kRowsAny ? a.cols : (a.cols + 7) / 8;
  auto fit = [&](int nc) { return ((chunks + nc - 1) / nc + 31) / 32 * 32; };
  const bool many = rows >= 8 * kNumSMs;
  if (layout == kRowsAligned) {
    if (fit(1) <= 512 && !(many && chunks >= 128)) return launch_add_norm<T, FP8, 8, 1, false, false>(a, rows, fit(1), st);
    if (fit(2) <= 512 && !(many && chunks >= 256)) return launch_add_norm<T, FP8, 8, 2, false, false>(a, rows, fit(2), st);
    if (fit(4) <= 512) return launch_add_norm<T, FP8, 8, 4, false, false>(a, rows, fit(4), st);
    return launch_add_norm<T, FP8, 8, 1, true, false>(a, rows, 512, st);
  }
  if (layout == kRowsShifted) {
    if (fit(1) <= 512 && !(many && chunks >= 128)) return launch_add_norm<T, FP8, 8, 1, false, true>(a, rows, fit(1), st);
    if (fit(4) <= 512) return launch_add_norm<T, FP8, 8, 4, false, true>(a, rows, fit(4), st);
  }
  // element by element
  const int t = (a.cols + 15) / 16 / 32 * 32 + 32;
  if (a.cols <= 2048) return launch_add_norm<T, FP8, 1, 4, false, false>(a, rows, ((a.cols + 3) / 4 + 31) / 32 * 32, st);
  if (t <= 512) return launch_add_norm<T, FP8, 1, 16, false, false>(a, rows, t, st);
  return launch_add_norm<T, FP8, 1, 1, true, false>(a, rows, 512, st);
}

bool vec_ok(const void* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride % 8) == 0;
}

}  // namespace
}  // namespace tv

using namespace tv;

extern "C" {

int tv_rms_norm(const void* x, int64_t x_row_stride, const void* weight, void* y, int64_t y_row_stride,
                int32_t rows, int32_t cols, float eps, int32_t dtype, void* stream) {
  if (rows < 0 || cols <= 0 || (cols % 8) != 0) return TV_ERR_SHAPE;
  if (dtype != TV_BF16 && dtype != TV_F16) return TV_ERR_DTYPE;
  if (rows == 0) return TV_OK;
  if (!x || !weight || !y) return TV_ERR_NULL;
  if (!vec_ok(x, x_row_stride) || !vec_ok(y, y_row_stride) || !vec_ok(weight, 0)) return TV_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TV_BF16)
    rms_norm_kernel<__nv_bfloat16><<<rows, kNormThreads, 0, st>>>(
        static_cast<const __nv_bfloat16*>(x), x_row_stride, static_cast<const __nv_bfloat16*>(weight),
        static_cast<__nv_bfloat16*>(y), y_row_stride, cols, eps);
  else
    rms_norm_kernel<__half><<<rows, kNormThreads, 0, st>>>(static_cast<const __half*>(x), x_row_stride,
                                                           static_cast<const __half*>(weight),
                                                           static_cast<__half*>(y), y_row_stride, cols, eps);
  return check_launch();
}

int tv_add_rms_norm(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride,
                    const void* weight, void* residual_out, int64_t residual_out_row_stride, void* y,
                    int64_t y_row_stride, float* y_scale, int32_t rows, int32_t cols, float eps, int32_t dtype,
                    void* stream) {
  if (rows < 0 || cols <= 0) return TV_ERR_SHAPE;
  if (dtype != TV_BF16 && dtype != TV_F16) return TV_ERR_DTYPE;
  if (cols > (1 << 30)) return TV_ERR_UNSUPPORTED;      // a thread's column index passes cols by up to 4096
  if (rows == 0) return TV_OK;
  if (!x || !residual || !weight || !residual_out || !y) return TV_ERR_NULL;
  AddNormArgs a{x, residual, weight, residual_out, y, y_scale, x_row_stride, residual_row_stride,
                residual_out_row_stride, y_row_stride, cols, eps};
  const bool y_ok = y_scale ? (reinterpret_cast<uintptr_t>(y) & 7) == 0 && (y_row_stride % 8) == 0
                            : vec_ok(y, y_row_stride);
  AddNormLayout layout = kRowsAny;
  // one row needs no stride of its own
  auto same = [&](const void* p, int64_t s) {
    return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0 &&
           (rows == 1 || ((s - x_row_stride) & 7) == 0);
  };
  if ((cols % 8) == 0 && vec_ok(x, x_row_stride) && vec_ok(residual, residual_row_stride) && vec_ok(weight, 0) &&
      vec_ok(residual_out, residual_out_row_stride) && y_ok)
    layout = kRowsAligned;
  else if (cols >= 64 && (reinterpret_cast<uintptr_t>(x) & 1) == 0 && same(residual, residual_row_stride) &&
           same(residual_out, residual_out_row_stride))
    layout = kRowsShifted;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TV_BF16)
    return y_scale ? pick_add_norm<__nv_bfloat16, true>(a, rows, layout, st)
                   : pick_add_norm<__nv_bfloat16, false>(a, rows, layout, st);
  return y_scale ? pick_add_norm<__half, true>(a, rows, layout, st)
                 : pick_add_norm<__half, false>(a, rows, layout, st);
}

int tv_silu_mul(const void* gate, const void* up, int64_t in_row_stride, void* out, int64_t out_row_stride,
                int32_t rows, int32_t cols, int32_t dtype, void* stream) {
  if (rows < 0 || cols <= 0 || (cols % 8) != 0) return TV_ERR_SHAPE;
  if (dtype != TV_BF16 && dtype != TV_F16) return TV_ERR_DTYPE;
  if (rows == 0) return TV_OK;
  if (!gate || !up || !out) return TV_ERR_NULL;
  if (!vec_ok(gate, in_row_stride) || !vec_ok(up, in_row_stride) || !vec_ok(out, out_row_stride))
    return TV_ERR_ALIGN;
  const int64_t n = (int64_t)rows * (cols / 8);
  const int threads = 256;
  const int64_t want = (n + threads - 1) / threads;
  const int blocks = (int)(want < 4 * kNumSMs ? want : 4 * kNumSMs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TV_BF16)
    silu_mul_kernel<__nv_bfloat16><<<blocks, threads, 0, st>>>(
        static_cast<const __nv_bfloat16*>(gate), static_cast<const __nv_bfloat16*>(up), in_row_stride,
        static_cast<__nv_bfloat16*>(out), out_row_stride, rows, cols);
  else
    silu_mul_kernel<__half><<<blocks, threads, 0, st>>>(static_cast<const __half*>(gate),
                                                        static_cast<const __half*>(up), in_row_stride,
                                                        static_cast<__half*>(out), out_row_stride, rows, cols);
  return check_launch();
}

}  // extern "C"
