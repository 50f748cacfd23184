// cawq_norm.cuh — RMS norm with the residual's addition (sm_100a).
//
//   h = x + r,  y = h / sqrt(mean(h^2) + eps) * w
//
// h stays in fp32 between the sum and y; y (and h, where it is written back)
// is rounded once. With FP8, y leaves as e4m3 of y / s, s = max |y| / 448 of
// its row.
#pragma once

#include <cuda_fp8.h>

#include "cawq_common.cuh"

namespace cawq {

constexpr int kNormThreads = 256;
constexpr float kE4m3Max = 448.f;

// Sum (or maximum) of one value per thread over the block; every thread gets it.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  const int warps = blockDim.x >> 5;
  __syncthreads();  // the scratch may still be read by an earlier reduction
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < warps; ++i) v = MAX ? fmaxf(v, scratch[i]) : v + scratch[i];
  return v;
}

template <int DT, bool FP8>
__global__ void __launch_bounds__(kNormThreads)
    rms_norm_kernel(const typename DType<DT>::T* x, const typename DType<DT>::T* __restrict__ w,
                    const typename DType<DT>::T* res, void* y, typename DType<DT>::T* res_out,
                    float* scales, uint32_t d, size_t ld_x, size_t ld_r, size_t ld_y, size_t ld_ro,
                    float eps) {
  using D = DType<DT>;
  using T = typename D::T;
  __shared__ float scratch[kNormThreads / 32];
  const size_t row = blockIdx.x;
  const T* xr = x + row * ld_x;
  const T* rr = res ? res + row * ld_r : nullptr;
  float sum = 0.f;
  for (uint32_t i = threadIdx.x; i < d; i += kNormThreads) {
    const float h = D::to_f32(xr[i]) + (rr ? D::to_f32(rr[i]) : 0.f);
    sum += h * h;
  }
  sum = block_reduce<false>(sum, scratch);
  const float rs = 1.f / sqrtf(sum / static_cast<float>(d) + eps);
  float inv = 0.f;
  if constexpr (FP8) {
    float top = 0.f;
    for (uint32_t i = threadIdx.x; i < d; i += kNormThreads) {
      const float h = D::to_f32(xr[i]) + (rr ? D::to_f32(rr[i]) : 0.f);
      top = fmaxf(top, fabsf(h * rs * D::to_f32(w[i])));
    }
    top = block_reduce<true>(top, scratch);
    inv = top > 0.f ? kE4m3Max / top : 0.f;
    if (threadIdx.x == 0) scales[row] = top / kE4m3Max;
  }
  for (uint32_t i = threadIdx.x; i < d; i += kNormThreads) {
    const float h = D::to_f32(xr[i]) + (rr ? D::to_f32(rr[i]) : 0.f);
    const float v = h * rs * D::to_f32(w[i]);
    if (res_out) res_out[row * ld_ro + i] = D::from_f32(h);
    if constexpr (FP8)
      static_cast<__nv_fp8_e4m3*>(y)[row * ld_y + i] = __nv_fp8_e4m3(v * inv);
    else
      static_cast<T*>(y)[row * ld_y + i] = D::from_f32(v);
  }
}

cudaError_t launch_rms_norm(const NormProblem& p) {
  const dim3 grid(static_cast<uint32_t>(p.rows));
#define CAWQ_NORM(DT, F8)                                                                      \
  rms_norm_kernel<DT, F8><<<grid, kNormThreads, 0, p.stream>>>(                               \
      static_cast<const DType<DT>::T*>(p.x), static_cast<const DType<DT>::T*>(p.w),           \
      static_cast<const DType<DT>::T*>(p.res), p.y, static_cast<DType<DT>::T*>(p.res_out),    \
      p.scales, static_cast<uint32_t>(p.d), p.ld_x, p.ld_res, p.ld_y, p.ld_res_out, p.eps)
  if (p.dtype == kF32) {
    if (p.scales) CAWQ_NORM(kF32, true); else CAWQ_NORM(kF32, false);
  } else if (p.dtype == kF16) {
    if (p.scales) CAWQ_NORM(kF16, true); else CAWQ_NORM(kF16, false);
  } else {
    if (p.scales) CAWQ_NORM(kBF16, true); else CAWQ_NORM(kBF16, false);
  }
#undef CAWQ_NORM
  return cudaGetLastError();
}

}  // namespace cawq
