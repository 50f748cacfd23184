// cawq_rope.cuh — rotary embedding of the new tokens' q and k, and the append
// of k and v to the paged cache, in one launch (sm_100a).
//
// Element i < D / 2 of a head turns with element i + D / 2 by the angle of the
// token's position: (a, b) -> (a c - b s, b c + a s), in fp32 with one
// rounding.
//
// Prompts (3083 tokens, 28 / 4 heads, bf16: 58 MB in 14.8 us, 3.9 TB/s) wait for
// the chain that each token's CTA goes through, sequence, length and row starts,
// page, angles, each load's address from the one before (5.3 cycles of long
// scoreboard stall an issue), beside 2-3 us of launch; single tokens are latency
// altogether (64 tokens, 32 / 32 heads, f16: 2.7 us). One CTA per token, a thread
// per 8 elements of the lower half of a head and the 8 that turn with them, so
// every access is 16 bytes; its loads go out before the token's sequence,
// position and page are looked up. (Two heads a thread, and CTAs of 128 or 256,
// were no faster: 14.6 and 17 us.)
#pragma once

#include "cawq_norm.cuh"
#include "cawq_paged.cuh"

namespace cawq {

constexpr int kRopeThreads = 1024;

template <int DT>
__global__ void __launch_bounds__(kRopeThreads)
    rope_append_kernel(const char* q, const char* k, const char* v, const float* __restrict__ rope,
                       char* q_out, const PagedView kv, uint32_t tokens, uint32_t n_q, uint32_t d,
                       uint32_t rope_rows, int64_t ld_q, int64_t ld_k, int64_t ld_v,
                       int64_t ld_qo) {
  using V = Vec16<DT>;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t t = blockIdx.x;
  const uint32_t shift = d == 64 ? 2 : 3;  // 4 or 8 threads a head
  const uint32_t items = (n_q + 2 * kv.n_kv) << shift;
  const uint32_t half = d;  // bytes of half a head
  auto source = [&](uint32_t i) {
    const uint32_t h = i >> shift, c = i & ((1u << shift) - 1);
    return (h < n_q ? q + t * ld_q + (int64_t)h * 2 * d
                    : h < n_q + kv.n_kv ? k + t * ld_k + (int64_t)(h - n_q) * 2 * d
                                        : v + t * ld_v + (int64_t)(h - n_q - kv.n_kv) * 2 * d) +
           16 * c;
  };
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (threadIdx.x < items) {
    const char* src = source(threadIdx.x);
    lo = *reinterpret_cast<const uint4*>(src);
    hi = *reinterpret_cast<const uint4*>(src + half);
  }
  // the position, while these loads are under way
  const uint32_t b = kv.sequence(t);
  int pos = -1;
  if (b < kv.batch) {
    int first, count;
    kv.rows(b, tokens, &first, &count);
    // a row before q_start[0], or one that starts out of order left outside its
    // sequence, has no place
    if (static_cast<int>(t) >= first && static_cast<int>(t) < first + count)
      pos = kv.len(b) - count + static_cast<int>(t) - first;
  }
  if (pos >= static_cast<int>(rope_rows)) {
    atomicOr(&g_cawq_device_error, kErrCache);
    pos = -1;
  }
  for (uint32_t i = threadIdx.x; i < items; i += blockDim.x) {
    const uint32_t h = i >> shift, c = i & ((1u << shift) - 1);
    if (i != threadIdx.x) {
      const char* src = source(i);
      lo = *reinterpret_cast<const uint4*>(src);
      hi = *reinterpret_cast<const uint4*>(src + half);
    }
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
    if (h < n_q + kv.n_kv) {
      float a[8], e[8], cs[8], sn[8];
      V::unpack(lo, a);
      V::unpack(hi, e);
      const float4* tab = reinterpret_cast<const float4*>(rope + (size_t)max(pos, 0) * d) + 2 * c;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = pos < 0 ? make_float4(0, 0, 0, 0) : __ldg(tab + j);
        const float4 y = pos < 0 ? make_float4(0, 0, 0, 0) : __ldg(tab + d / 8 + j);
        cs[4 * j] = x.x, cs[4 * j + 1] = x.y, cs[4 * j + 2] = x.z, cs[4 * j + 3] = x.w;
        sn[4 * j] = y.x, sn[4 * j + 1] = y.y, sn[4 * j + 2] = y.z, sn[4 * j + 3] = y.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = a[j] * cs[j] - e[j] * sn[j], w = e[j] * cs[j] + a[j] * sn[j];
        a[j] = pos < 0 ? 0.f : u;  // a token of no place: zeros, whatever q holds
        e[j] = pos < 0 ? 0.f : w;
      }
      lo = V::pack(a);
      hi = V::pack(e);
    }
    *reinterpret_cast<uint4*>(dst + 16 * c) = lo;
    *reinterpret_cast<uint4*>(dst + half + 16 * c) = hi;
  }
}

cudaError_t launch_rope_append(const RopeProblem& p, const PagedView& kv) {
  const char *q = static_cast<const char*>(p.q), *k = static_cast<const char*>(p.k);
  const char* v = static_cast<const char*>(p.v);
  const float* rope = p.rope;
  char* q_out = static_cast<char*>(p.q_out);
  PagedView view = kv;
  uint32_t tokens = static_cast<uint32_t>(p.tokens), n_q = static_cast<uint32_t>(p.n_q);
  uint32_t d = static_cast<uint32_t>(p.d), rope_rows = static_cast<uint32_t>(p.rope_rows);
  int64_t ld_q = (int64_t)p.ld_q * 2, ld_k = (int64_t)p.ld_k * 2, ld_v = (int64_t)p.ld_v * 2;
  int64_t ld_qo = (int64_t)p.ld_q_out * 2;
  void* a[] = {&q, &k, &v, &rope, &q_out, &view, &tokens, &n_q, &d, &rope_rows, &ld_q, &ld_k,
               &ld_v, &ld_qo};
  // a thread per item where a CTA has room for a token's
  const uint32_t items = (n_q + 2 * kv.n_kv) * (d / 16);
  const int threads = static_cast<int>(std::min<uint32_t>((items + 31) / 32 * 32, kRopeThreads));
  return launch_pdl(p.dtype == kF16 ? rope_append_kernel<kF16> : rope_append_kernel<kBF16>,
                    dim3(tokens), threads, 0, p.stream, a);
}

}  // namespace cawq
