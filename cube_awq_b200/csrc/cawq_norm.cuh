// cawq_norm.cuh — RMS norm with the residual's addition (sm_100a).
//
//   h = x + r,  y = h / sqrt(mean(h^2) + eps) * w
//
// h stays in fp32 between the sum and y; y (and h, where it is written back)
// is rounded once. With FP8, y leaves as e4m3 of y / s, s = max |y| / 448 of
// its row.
//
// Bound by bytes: x, r and h once, y once. A row's h stays in registers
// between the passes over it, 16-byte vectors, VPT of them a thread, so every
// byte moves once. Rows of up to 32 vectors x 4 take a warp each (8 rows a CTA),
// longer ones a CTA. Few rows are latency: one vector a thread (the row's
// loads all go out at once); many rows are bandwidth: four a thread, so that
// an SM holds more rows at a time (4099 x 8192 with the residual: bf16 42.4 us,
// 6.3 TB/s; bf16 to e4m3 41.5-41.9 us, 5.6 TB/s; f32, eight vectors a thread, 81.4
// us, 6.6 TB/s; 1 x 4096 f16 2.2 us). Rows off 16-byte alignment go
// element by element, still in registers up to 16384 elements, and longer ones
// through the caches again in each pass.
#pragma once

#include <cuda_fp8.h>

#include "cawq_common.cuh"

namespace cawq {

constexpr int kNormThreads = 256;  // of CTAs with a row a warp, and for the longest rows
constexpr float kE4m3Max = 448.f;
// Below this largest |y| of a row (448 / FLT_MAX is 1.3e-36) 448 / max |y| may
// pass fp32's range: y and the maximum are multiplied by 2^64 first, exactly.
constexpr float kTinyTop = 0x1p-118f, kTinyUp = 0x1p64f;

// The larger one, NaN where either is (fmaxf would pass it by).
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum (or maximum) of one value per thread over the block; every thread gets it.
template <bool MAX>
__device__ __forceinline__ float warp_reduce(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_or_nan(v, u) : v + u;
  }
  return v;
}
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* scratch) {
  v = warp_reduce<MAX>(v);
  const int warps = blockDim.x >> 5;
  __syncthreads();  // the scratch may still be read by an earlier reduction
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < warps; ++i) v = MAX ? max_or_nan(v, scratch[i]) : v + scratch[i];
  return v;
}

template <int DT>
struct NormArgs {
  using T = typename DType<DT>::T;
  const T *x, *w, *res;  // res, res_out: may be null; they and y may alias x / res row by row
  void* y;
  T* res_out;
  float* scales;
  uint32_t rows, d;
  size_t ld_x, ld_r, ld_y, ld_ro;
  float eps;
};

// Element by element; EPT elements of the row stay with a thread, or none
// (EPT 0: rows of any length, read again in each pass).
template <int DT, bool FP8, int EPT>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs<DT> a) {
  using D = DType<DT>;
  using T = typename D::T;
  constexpr int N = EPT > 0 ? EPT : 1;
  __shared__ float scratch[32];
  pdl_wait();
  pdl_launch_dependents();
  const size_t row = blockIdx.x;
  const T* xr = a.x + row * a.ld_x;
  const T* rr = a.res ? a.res + row * a.ld_r : nullptr;
  auto sum_at = [&](uint32_t i) { return D::to_f32(xr[i]) + (rr ? D::to_f32(rr[i]) : 0.f); };
  float h[N], sum = 0.f;
  // f(i, h of element i) for this thread's elements
  auto each = [&](auto f) {
    if constexpr (EPT > 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint32_t i = threadIdx.x + k * blockDim.x;
        if (i < a.d) f(i, h[k]);
      }
    } else {
      for (uint32_t i = threadIdx.x; i < a.d; i += blockDim.x) f(i, sum_at(i));
    }
  };
  if constexpr (EPT > 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t i = threadIdx.x + k * blockDim.x;
      h[k] = i < a.d ? sum_at(i) : 0.f;
    }
  }
  each([&](uint32_t, float v) { sum += v * v; });
  sum = block_reduce<false>(sum, scratch);
  const float rs = 1.f / sqrtf(sum / static_cast<float>(a.d) + a.eps);
  float inv = 0.f, up = 1.f;
  if constexpr (FP8) {
    float top = 0.f;
    each([&](uint32_t i, float v) { top = max_or_nan(top, fabsf(v * rs * D::to_f32(a.w[i]))); });
    top = block_reduce<true>(top, scratch);
    if (threadIdx.x == 0) a.scales[row] = top / kE4m3Max;
    if (top < kTinyTop) up = kTinyUp;
    inv = top > 0.f ? kE4m3Max / (top * up) : 0.f;
  }
  each([&](uint32_t i, float u) {
    const float v = u * rs * D::to_f32(a.w[i]);
    if (a.res_out) a.res_out[row * a.ld_ro + i] = D::from_f32(u);
    if constexpr (FP8)
      static_cast<__nv_fp8_e4m3*>(a.y)[row * a.ld_y + i] = __nv_fp8_e4m3(v * up * inv);
    else
      static_cast<T*>(a.y)[row * a.ld_y + i] = D::from_f32(v);
  });
}

// 16 bytes as fp32 values and back
template <int DT>
struct Vec16 {
  using T = typename DType<DT>::T;
  static constexpr int kN = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[kN]) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < kN; ++i) f[i] = DType<DT>::to_f32(e[i]);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[kN]) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < kN; ++i) e[i] = DType<DT>::from_f32(f[i]);
    return u;
  }
};

// WARP: a row a warp; else a row a CTA.
template <int DT, bool FP8, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP || VPT == 4 ? kNormThreads : VPT == 1 ? 1024 : 512,
                                  VPT == 4 ? 3 : 1)  // three: 80 registers
    rms_norm_vec_kernel(const NormArgs<DT> a) {
  using V = Vec16<DT>;
  constexpr int N = V::kN;
  __shared__ float scratch[32];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t lane = WARP ? threadIdx.x & 31 : threadIdx.x;
  const uint32_t step = WARP ? 32 : blockDim.x;
  const size_t row = WARP ? static_cast<size_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)
                          : blockIdx.x;
  if (WARP && row >= a.rows) return;
  const uint32_t nv = a.d / N;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ld_x);
  const uint4* rr = reinterpret_cast<const uint4*>(a.res + row * a.ld_r);
  const uint4* wr = reinterpret_cast<const uint4*>(a.w);
  auto reduce = [&](float v, auto max) {
    if constexpr (WARP) return warp_reduce<decltype(max)::value>(v);
    else return block_reduce<decltype(max)::value>(v, scratch);
  };
  uint4 ux[VPT], ur[VPT], uw[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t v = lane + i * step;
    if (v < nv) {
      ux[i] = xr[v];
      if (a.res) ur[i] = rr[v];
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (lane + i * step < nv) uw[i] = __ldg(wr + lane + i * step);
  float h[VPT][N], sum = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (lane + i * step < nv) {
      V::unpack(ux[i], h[i]);
      if (a.res) {
        float r[N];
        V::unpack(ur[i], r);
#pragma unroll
        for (int k = 0; k < N; ++k) h[i][k] += r[k];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) sum += h[i][k] * h[i][k];
    }
  }
  sum = reduce(sum, std::false_type{});
  const float rs = 1.f / sqrtf(sum / static_cast<float>(a.d) + a.eps);
  if (a.res_out) {
    uint4* o = reinterpret_cast<uint4*>(a.res_out + row * a.ld_ro);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (lane + i * step < nv) o[lane + i * step] = V::pack(h[i]);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (lane + i * step < nv) {
      float w[N];
      V::unpack(uw[i], w);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        h[i][k] = h[i][k] * rs * w[k];
        if constexpr (FP8) top = max_or_nan(top, fabsf(h[i][k]));
      }
    }
  }
  if constexpr (FP8) {
    top = reduce(top, std::true_type{});
    if (lane == 0) a.scales[row] = top / kE4m3Max;
    if (top < kTinyTop) {
      top *= kTinyUp;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k) h[i][k] *= kTinyUp;
    }
    const float inv = top > 0.f ? kE4m3Max / top : 0.f;
    uint8_t* o = static_cast<uint8_t*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t v = lane + i * step;
      if (v < nv) {
        uint32_t b[N / 4];
#pragma unroll
        for (int k = 0; k < N; k += 4) {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(
              make_float2(h[i][k] * inv, h[i][k + 1] * inv), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(
              make_float2(h[i][k + 2] * inv, h[i][k + 3] * inv), __NV_SATFINITE, __NV_E4M3);
          b[k / 4] = lo | hi << 16;
        }
        if constexpr (N == 8)
          *reinterpret_cast<uint2*>(o + 8 * v) = make_uint2(b[0], b[1]);
        else
          *reinterpret_cast<uint32_t*>(o + 4 * v) = b[0];
      }
    }
  } else {
    uint4* o = reinterpret_cast<uint4*>(static_cast<typename NormArgs<DT>::T*>(a.y) + row * a.ld_y);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (lane + i * step < nv) o[lane + i * step] = V::pack(h[i]);
  }
}

template <int DT, bool FP8>
cudaError_t launch_rms_norm_t(const NormProblem& p) {
  using T = typename DType<DT>::T;
  NormArgs<DT> a = {static_cast<const T*>(p.x), static_cast<const T*>(p.w),
                    static_cast<const T*>(p.res), p.y, static_cast<T*>(p.res_out), p.scales,
                    static_cast<uint32_t>(p.rows), static_cast<uint32_t>(p.d), p.ld_x, p.ld_res,
                    p.ld_y, p.ld_res_out, p.eps};
  constexpr size_t N = Vec16<DT>::kN;
  void* args[] = {&a};
  auto vec = [](const void* q, size_t ld, size_t bytes) {
    return !q || (reinterpret_cast<uintptr_t>(q) % bytes == 0 && ld % N == 0);
  };
  const bool fits = p.d % N == 0 && p.d / N <= 8 * 512 && vec(p.x, p.ld_x, 16) &&
                    vec(p.res, p.ld_res, 16) && vec(p.res_out, p.ld_res_out, 16) &&
                    vec(p.w, 0, 16) && vec(p.y, p.ld_y, FP8 ? N : 16);
  const uint32_t rows = static_cast<uint32_t>(p.rows);
  if (!fits) {
    const uint32_t ept = p.d <= 8 * 1024 ? 8 : 16;
    const int few = static_cast<int>(((p.d + ept - 1) / ept + 31) / 32 * 32);
    if (p.d > 16 * 1024)
      return launch_pdl(rms_norm_kernel<DT, FP8, 0>, dim3(rows), kNormThreads, 0, p.stream, args);
    return ept == 8
               ? launch_pdl(rms_norm_kernel<DT, FP8, 8>, dim3(rows), few, 0, p.stream, args)
               : launch_pdl(rms_norm_kernel<DT, FP8, 16>, dim3(rows), few, 0, p.stream, args);
  }
  const uint32_t nv = static_cast<uint32_t>(p.d / N);
  auto threads = [&](uint32_t vpt) { return static_cast<int>(((nv + vpt - 1) / vpt + 31) / 32 * 32); };
  const bool many = rows >= 2u * p.sm_count;
  if (nv <= 32 * 4 && many) {
    constexpr uint32_t R = kNormThreads / 32;
    const dim3 grid((rows + R - 1) / R);
    if (nv <= 32)
      return launch_pdl(rms_norm_vec_kernel<DT, FP8, 1, true>, grid, kNormThreads, 0, p.stream, args);
    return launch_pdl(rms_norm_vec_kernel<DT, FP8, 4, true>, grid, kNormThreads, 0, p.stream, args);
  }
  if (!many && nv <= 1024)
    return launch_pdl(rms_norm_vec_kernel<DT, FP8, 1, false>, dim3(rows), threads(1), 0, p.stream,
                      args);
  if (nv <= 4 * kNormThreads)
    return launch_pdl(rms_norm_vec_kernel<DT, FP8, 4, false>, dim3(rows), threads(4), 0, p.stream,
                      args);
  return launch_pdl(rms_norm_vec_kernel<DT, FP8, 8, false>, dim3(rows), threads(8), 0, p.stream,
                    args);
}

cudaError_t launch_rms_norm(const NormProblem& p) {
#define CAWQ_NORM(DT) (p.scales ? launch_rms_norm_t<DT, true>(p) : launch_rms_norm_t<DT, false>(p))
  return p.dtype == kF32 ? CAWQ_NORM(kF32) : p.dtype == kF16 ? CAWQ_NORM(kF16) : CAWQ_NORM(kBF16);
#undef CAWQ_NORM
}

}  // namespace cawq
