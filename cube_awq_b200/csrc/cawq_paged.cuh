// cawq_paged.cuh — the paged key / value cache as the layer kernels see it:
// which sequence a new token belongs to, its position, and where a position
// lies in the cache. All values that come from device memory (lengths, row
// starts, page numbers) are bounded here, so no value of theirs makes a kernel
// read or write outside its buffers; what is skipped sets bit 2 of the device
// error word.
#pragma once

#include "cawq_common.cuh"

namespace cawq {

constexpr uint32_t kErrCache = 4u;  // bit 2 of the device error word

// n / d and n % d for n < 2^31: q = (n * m) >> (31 + s) with s = ceil(log2 d),
// m = ceil(2^(31 + s) / d). The error n * (m d - 2^(31+s)) / (d 2^(31+s)) is
// below 2^31 * 2^s / (d 2^(31+s)) <= 1 / d, so the floor is exact.
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t v = 1) : d(v), s(0) {
    while ((1ull << s) < v) ++s;
    m = static_cast<uint32_t>(((1ull << (31 + s)) + v - 1) / v);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> (31 + s));
  }
};

struct PagedView {
  char* k;
  char* v;
  int64_t sp, sh, st;  // page, head and token strides in bytes
  const int32_t* table;
  const int32_t* lens;
  const int32_t* q_start;  // nullptr: one new token per sequence
  int64_t ld_table;
  uint32_t pages, width, batch, n_kv;
  FastDiv page;

  // positions that a table row can hold
  __device__ __forceinline__ int cap() const { return static_cast<int>(width * page.d); }
  // tokens of sequence b. More than cap() of them set the error bit: the new
  // tokens' positions follow from the length as it is, keys end at cap().
  __device__ __forceinline__ int len(uint32_t b) const {
    const int n = lens[b];
    if (n > cap()) atomicOr(&g_cawq_device_error, kErrCache);
    return max(0, n);
  }
  // rows [first, first + count) of the call's tensors are sequence b's
  __device__ __forceinline__ void rows(uint32_t b, uint32_t tokens, int* first, int* count) const {
    if (!q_start) {
      *first = static_cast<int>(b);
      *count = 1;
      return;
    }
    const int a = max(0, min(q_start[b], static_cast<int>(tokens)));
    const int e = max(a, min(q_start[b + 1], static_cast<int>(tokens)));
    *first = a;
    *count = e - a;
  }
  // the sequence of row t (batch if none): how many q_start[b + 1] are <= t,
  // by a search that a whole warp makes with 32 probes a step. Row t may lie
  // outside rows(b) all the same: before q_start[0], or where q_start does not
  // ascend.
  __device__ __forceinline__ uint32_t sequence(uint32_t t) const {
    if (!q_start) return t;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, span = batch;
    for (;;) {
      const uint32_t step = (span + 31) / 32, at = lo + (lane + 1) * step - 1;
      const bool past = (lane + 1) * step <= span && q_start[at + 1] <= static_cast<int>(t);
      lo += __popc(__ballot_sync(0xffffffffu, past)) * step;
      if (step <= 1) return lo;
      span = min(step, batch - lo);
    }
  }
  // byte offset of position j of sequence b, head h (the same in k and v);
  // -1 (and the error bit) if its page is past the table or none of the cache's.
  __device__ __forceinline__ int64_t offset(uint32_t b, uint32_t h, uint32_t j) const {
    const uint32_t p = page.div(j);
    const int32_t pg = p < width ? table[b * ld_table + p] : -1;
    if (static_cast<uint32_t>(pg) >= pages) {
      atomicOr(&g_cawq_device_error, kErrCache);
      return -1;
    }
    return pg * sp + h * sh + static_cast<int64_t>(j - p * page.d) * st;
  }
};

}  // namespace cawq
