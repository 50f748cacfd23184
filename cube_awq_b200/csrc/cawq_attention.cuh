// cawq_attention.cuh — attention of new tokens over a paged cache (sm_100a).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// over the visible positions, m their running maximum. One warp per (token,
// query head); the lanes hold the head's dimensions and the keys pass one by
// one.
#pragma once

#include "cawq_paged.cuh"

namespace cawq {

template <int DT, int D>
__global__ void __launch_bounds__(128)
    attention_kernel(const char* q, char* out, const PagedView kv, uint32_t tokens, uint32_t n_q,
                     int64_t ld_q, int64_t ld_o, float scale_log2, int window, int sinks) {
  using T = typename DType<DT>::T;
  constexpr int E = D / 32;
  const uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (uint64_t)tokens * n_q) return;
  const uint32_t t = static_cast<uint32_t>(w / n_q), h = static_cast<uint32_t>(w % n_q);
  const int lane = threadIdx.x & 31;
  const uint32_t b = kv.sequence(t);
  if (b >= kv.batch) return;
  int first, count;
  kv.rows(b, tokens, &first, &count);
  const int pos = kv.len(b) - count + static_cast<int>(t) - first;
  const uint32_t hk = h / (n_q / kv.n_kv);
  float qf[E], o[E];
  const T* qr = reinterpret_cast<const T*>(q + t * ld_q + (int64_t)h * D * 2) + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qf[i] = DType<DT>::to_f32(qr[i]) * scale_log2;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int start = window > 0 ? max(0, pos - window + 1) : 0;
  for (int j = start > 0 && sinks > 0 ? 0 : start; j <= pos; ++j) {
    if (j >= sinks && j < start) j = start;
    const int64_t at = kv.offset(b, hk, static_cast<uint32_t>(j));
    if (at < 0) continue;
    const T* kr = reinterpret_cast<const T*>(kv.k + at) + lane * E;
    const T* vr = reinterpret_cast<const T*>(kv.v + at) + lane * E;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += qf[i] * DType<DT>::to_f32(kr[i]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float c = exp2f(m - base), p = exp2f(s - base);
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * c + p * DType<DT>::to_f32(vr[i]);
    m = mn;
  }
  T* orow = reinterpret_cast<T*>(out + t * ld_o + (int64_t)h * D * 2) + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) orow[i] = DType<DT>::from_f32(l != 0.f ? o[i] / l : 0.f);
}

cudaError_t launch_attention(const AttentionProblem& p, const PagedView& kv) {
  const dim3 grid(static_cast<uint32_t>((p.tokens * p.n_q + 3) / 4));
#define CAWQ_ATT(DT, D)                                                                        \
  attention_kernel<DT, D><<<grid, 128, 0, p.stream>>>(                                         \
      static_cast<const char*>(p.q), static_cast<char*>(p.out), kv,                            \
      static_cast<uint32_t>(p.tokens), static_cast<uint32_t>(p.n_q), (int64_t)p.ld_q * 2,      \
      (int64_t)p.ld_out * 2, p.scale * 1.4426950408889634f, p.window, p.sinks)
  if (p.dtype == kF16) {
    if (p.d == 64) CAWQ_ATT(kF16, 64); else CAWQ_ATT(kF16, 128);
  } else {
    if (p.d == 64) CAWQ_ATT(kBF16, 64); else CAWQ_ATT(kBF16, 128);
  }
#undef CAWQ_ATT
  return cudaGetLastError();
}

}  // namespace cawq
