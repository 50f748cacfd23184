// cawq_rope.cuh — rotary embedding of the new tokens' q and k, and the append
// of k and v to the paged cache, in one launch (sm_100a).
//
// Element i < D / 2 of a head turns with element i + D / 2 by the angle of the
// token's position: (a, b) -> (a c - b s, b c + a s), in fp32 with one
// rounding. One CTA per token; a thread takes 8 elements of the lower half and
// the 8 that turn with them, so every access is 16 bytes.
#pragma once

#include "cawq_paged.cuh"

namespace cawq {

constexpr int kRopeThreads = 256;

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  using T = typename DType<DT>::T;
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = DType<DT>::to_f32(e[i]);
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  using T = typename DType<DT>::T;
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = DType<DT>::from_f32(f[i]);
  return u;
}

template <int DT>
__global__ void __launch_bounds__(kRopeThreads)
    rope_append_kernel(const char* q, const char* k, const char* v, const float* __restrict__ rope,
                       char* q_out, const PagedView kv, uint32_t tokens, uint32_t n_q, uint32_t d,
                       uint32_t rope_rows, int64_t ld_q, int64_t ld_k, int64_t ld_v,
                       int64_t ld_qo) {
  const uint32_t t = blockIdx.x;
  const uint32_t b = kv.sequence(t);
  int pos = -1;
  if (b < kv.batch) {
    int first, count;
    kv.rows(b, tokens, &first, &count);
    pos = kv.len(b) - count + static_cast<int>(t) - first;
  }
  if (pos >= static_cast<int>(rope_rows)) {
    atomicOr(&g_cawq_device_error, kErrCache);
    pos = -1;
  }
  const uint32_t per = d / 16;  // threads a head takes
  const uint32_t items = (n_q + 2 * kv.n_kv) * per;
  const uint32_t half = d;  // bytes of half a head
  for (uint32_t i = threadIdx.x; i < items; i += kRopeThreads) {
    const uint32_t h = i / per, c = i - h * per;
    const char* src = h < n_q ? q + t * ld_q + (int64_t)h * 2 * d
                      : h < n_q + kv.n_kv ? k + t * ld_k + (int64_t)(h - n_q) * 2 * d
                                          : v + t * ld_v + (int64_t)(h - n_q - kv.n_kv) * 2 * d;
    char* dst;
    if (h < n_q) {
      dst = q_out + t * ld_qo + (int64_t)h * 2 * d;
    } else {
      if (pos < 0) continue;
      const bool is_v = h >= n_q + kv.n_kv;
      const int64_t at = kv.offset(b, h - n_q - (is_v ? kv.n_kv : 0), static_cast<uint32_t>(pos));
      if (at < 0) continue;
      dst = (is_v ? kv.v : kv.k) + at;
    }
    uint4 lo = *reinterpret_cast<const uint4*>(src + 16 * c);
    uint4 hi = *reinterpret_cast<const uint4*>(src + half + 16 * c);
    if (h < n_q + kv.n_kv) {
      float a[8], e[8];
      unpack8<DT>(lo, a);
      unpack8<DT>(hi, e);
      const float* cs = rope + (size_t)(pos < 0 ? 0 : pos) * d + 8 * c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = pos < 0 ? 0.f : cs[j], y = pos < 0 ? 0.f : cs[d / 2 + j];
        const float u = a[j] * x - e[j] * y, w = e[j] * x + a[j] * y;
        a[j] = pos < 0 ? 0.f : u;
        e[j] = pos < 0 ? 0.f : w;
      }
      lo = pack8<DT>(a);
      hi = pack8<DT>(e);
    }
    *reinterpret_cast<uint4*>(dst + 16 * c) = lo;
    *reinterpret_cast<uint4*>(dst + half + 16 * c) = hi;
  }
}

cudaError_t launch_rope_append(const RopeProblem& p, const PagedView& kv) {
  const dim3 grid(static_cast<uint32_t>(p.tokens));
#define CAWQ_ROPE(DT)                                                                           \
  rope_append_kernel<DT><<<grid, kRopeThreads, 0, p.stream>>>(                                 \
      static_cast<const char*>(p.q), static_cast<const char*>(p.k),                            \
      static_cast<const char*>(p.v), p.rope, static_cast<char*>(p.q_out), kv,                  \
      static_cast<uint32_t>(p.tokens), static_cast<uint32_t>(p.n_q),                           \
      static_cast<uint32_t>(p.d), static_cast<uint32_t>(p.rope_rows), (int64_t)p.ld_q * 2,     \
      (int64_t)p.ld_k * 2, (int64_t)p.ld_v * 2, (int64_t)p.ld_q_out * 2)
  if (p.dtype == kF16) CAWQ_ROPE(kF16); else CAWQ_ROPE(kBF16);
#undef CAWQ_ROPE
  return cudaGetLastError();
}

}  // namespace cawq
