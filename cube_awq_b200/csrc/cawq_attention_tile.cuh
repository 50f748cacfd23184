// cawq_attention_tile.cuh — attention of many query rows over a paged cache on
// the 5th-generation tensor cores (sm_100a): prompts and chunks of prompts.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (q . k_j) - m),  c = scale log2(e)
//
// over the visible positions j of the row.
//
// Bound by the tensor cores: 4 D operations per (row, visible key). Measured,
// D = 128: 8192 tokens, 32 / 8 heads, f16, 532-540 us = 1020-1030 TFLOP/s
// sustained, where the GPU's power cap (1000 W) holds the clock at 1.5 GHz, and
// 452-474 us in short bursts; a chunk of 2048 tokens under a window of 4096, 64 /
// 8 heads, bf16, 319 us sustained, 282-320 in bursts; 7 ragged prompts, 28 / 4
// heads, bf16, 70-92 us.
//
// A CTA takes 256 query rows of one (sequence, kv head), as two halves of 128
// (one, where that leaves half the SMs idle):
// the rows are the G = n_q / n_kv query heads of consecutive tokens, token by
// token, so the heads that share keys share their loads whatever G is, and the
// key blocks of 128 that the causal mask or the window cut are few. Warps:
//   0-7, 8-15 softmax of half 0 and 1: 16 rows a warp, four threads a row
//             (with a row a thread and four warps a half a block took 2400
//             cycles, most of them latency; the tensor cores need 1024)
//   16, 17    tensor memory; one thread each issues the score products and the
//             second products (one for both spent its waits and commits one
//             after the other while the tensor cores idled). The whole warp
//             runs the loop and only the instruction is one thread's, which
//             keeps descriptors in uniform registers: otherwise an MMA took
//             126 cycles to issue, twice what it takes to run
//   18, 19    K_j and V_j of block j through one ring of 128-key stages (TMA,
//             128-byte swizzle; a box is a page's keys, or a power of two of
//             them that divides the page)
// Tensor memory: one slot for the scores S of a block and half (128 fp32
// columns), the weights P_0, P_1 (64 columns, the operand type), O_0, O_1 (D
// fp32 columns each). P is the A operand of the second product from there; V,
// which lies key by key, its MN-major B operand. The softmax warps move S to
// registers at once and free the slot, so that the halves take turns with it
// and a half's softmax of one block runs while the tensor cores do three
// products, its own next scores among them. (With S_h and P_h in one place,
// S_h(j + 1) had to wait for PV_h(j), and a block took the softmax and two
// products.)
//
// One CTA per tile: a grid of one CTA per SM whose roles ran on from tile to
// tile was slower (8192 tokens 530 against 495 us, ragged prompts 150 against
// 101 us on one GPU), as were two threads a row that trade their maxima, and
// exponentials on the FMA pipe for part of the weights (the loop waits for
// hand-overs and instruction slots, not for the special-function unit).
//
// The running maximum and sum are those of the online softmax (M. Milakov and N.
// Gimelshein, "Online normalizer calculation for softmax", 2018), in its
// published variant with a threshold: m moves only when a row's block maximum
// exceeds it by more than 2^8: p stays below 2^8 either way, nothing overflows (the sums are
// fp32, f16 holds 65504), and the row's O is rescaled a few times per row
// instead of once per block. It does so once PV(j - 1) has been added. The
// weights are rounded to the operand type, which is what the second product
// takes, and their sum is of the unrounded ones: against 64 bits the output's
// error is 2.1e-3 to 2.3e-3 in bf16 and 2.6e-4 in f16 (relative, ragged and
// windowed prompts, 8192 tokens), where weights of 32 bits leave 1.6e-3 to
// 1.7e-3 and 2.0e-4.
//
// Stale memory. Pages that no row of the tile needs (past the end, before the
// window) are not read: their boxes are requested outside the tensor and
// arrive as zeros. The last page's rows past the end may hold anything; for K
// they only reach masked scores, for V the box is written row by row with
// zeros past the end, since 0 * NaN is NaN. What is loaded for some rows and
// masked for others has weight 0 there and must be finite. A page number
// outside the cache hides its keys (s_bad) and sets the error bit.
//
// Every wait is bounded (2 s); on a timeout the kernel sets bit 0 of the
// device error word, stops issuing, waits (bounded) for what it issued, frees
// its TMEM and returns.
#pragma once

#include "cawq_attention.cuh"
#include "cawq_tcgen05.cuh"

namespace cawq {

constexpr uint32_t kTileRows = 256;  // or half of them (launch_attention_tile_t)
constexpr int kTileKeys = 128;
constexpr int kTileThreads = 640;
constexpr int kTileLoaders = 2;  // warps that issue the loads of a stage
constexpr float kTileSlack = 8.f;  // log2 of how far a row's maximum may be exceeded

template <int D>
struct TileLayout {
  static constexpr int kHalf = 128 * D * 2;  // 128 rows of q, or keys, or values
  static constexpr int kBlk = 128 * 128;     // of q: a 64-element column block
  static constexpr int kGroup = 8 * D * 2;   // of keys, values: 8 of them, by column blocks
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kOffKV = 2 * kHalf;
  static constexpr int kOffBars = kOffKV + kStages * kHalf;
  static constexpr int kSmem = 1024 + kOffBars + 512;
};

// Two fp32 values in one register pair: sm_100's packed arithmetic.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 4 x 4 transpose among four neighbouring lanes: v[k] of lane t -> v[t] of lane k.
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[4], int t) {
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {  // exchange with lane t ^ d
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k & d) continue;
      const uint32_t give = t & d ? v[k] : v[k | d];
      const uint32_t got = __shfl_xor_sync(0xffffffffu, give, d);
      if (t & d) v[k] = got; else v[k | d] = got;
    }
  }
}

// n ones from bit 0 on, for any n
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

struct TileArgs {
  const char* q;
  char* out;
  AttWork w;
  int64_t ld_q, ld_o;
  float scale_log2;   // > 0
  uint32_t negate;    // the score product's "negate A" bit with a negative scale
  uint32_t box;       // keys of a TMA box: divides page size and 128, a multiple of 8
  int64_t heads_per_page;  // page stride / head stride
};

// Stages of a tile in the producers' order: K_0, then K_{j+1}, V_j.
__device__ __forceinline__ uint32_t tile_stage_k(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ uint32_t tile_stage_v(int j, int nb) {
  return j + 1 < nb ? 2 * j + 2 : 2 * nb - 1;
}

// A CTA's tile: its sequence (0xffffffff: none), which of the sequence's tiles,
// and what the sequence has.
struct TilePick {
  uint32_t seq, tile;
  int first, count, len;
};

// few: the split kernel takes the sequences of few rows
__device__ __forceinline__ uint32_t tile_count(const AttWork& w, int count, bool few) {
  const uint32_t rows = static_cast<uint32_t>(count) * w.group;
  return few && rows <= kAttFewRows ? 0u : (rows + w.row_tile - 1) / w.row_tile;
}

// Tile number `index` of up to 32 sequences, longest first: lane b counts the
// tiles of sequence b whose last row is at key block v or later, and v is found
// by bisection. (Sequence by sequence, one of 2545 tokens after one of 2900
// began when the first was nearly done: a batch of 7 prompts 95 us, so 73.)
__device__ __forceinline__ TilePick pick_tile(const AttWork& w, uint32_t index) {
  const uint32_t lane = threadIdx.x & 31;
  TilePick t = {lane, 0, 0, 0, 0};
  if (lane < w.kv.batch) {
    w.kv.rows(lane, w.tokens, &t.first, &t.count);
    t.len = w.kv.len(lane);
  }
  const bool few = w.shared && AttLoad::of(w, t.count, t.len).of_warp().splits();
  const uint32_t tiles = tile_count(w, t.count, few);
  uint32_t n = tiles;
  const uint32_t total = __reduce_add_sync(0xffffffffu, n);
  if (index >= total) return {0xffffffffu, 0, 0, 0, 0};
  uint32_t at = index;  // among the tiles of the chosen block
  uint32_t later = 0;   // this sequence's tiles past it
  if (w.kv.batch > 1) {
    const int64_t rows = static_cast<int64_t>(t.count) * w.group;
    auto reach = [&](int v) -> uint32_t {  // tiles whose last row's position is >= 128 v
      if (n == 0) return 0;
      const int64_t row = (static_cast<int64_t>(v) * kTileKeys - (t.len - t.count)) * w.group;
      if (row <= 0) return n;
      return row >= rows ? 0u : n - static_cast<uint32_t>(row / w.row_tile);
    };
    int lo = 0, hi = static_cast<int>(__reduce_max_sync(0xffffffffu, n ? t.len : 0)) / kTileKeys + 1;
    while (hi - lo > 1) {  // the largest block that still has `index` tiles before or in it
      const int mid = (lo + hi) >> 1;
      if (__reduce_add_sync(0xffffffffu, reach(mid)) > index) lo = mid; else hi = mid;
    }
    later = reach(lo + 1);
    at -= __reduce_add_sync(0xffffffffu, later);
    n = (lo > 0 ? reach(lo) : n) - later;
  }
  uint32_t inc = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= static_cast<uint32_t>(o)) inc += v;
  }
  const int from = __ffs(__ballot_sync(0xffffffffu, at < inc)) - 1;
  t.tile = tiles - 1 - (later + at - (inc - n));
  t.seq = from;
  t.tile = __shfl_sync(0xffffffffu, t.tile, from);
  t.first = __shfl_sync(0xffffffffu, t.first, from);
  t.count = __shfl_sync(0xffffffffu, t.count, from);
  t.len = __shfl_sync(0xffffffffu, t.len, from);
  return t;
}

// The same of any number of sequences, sequence by sequence, the last tile of
// each first. All threads; the result is in *pick after the next barrier.
__device__ __forceinline__ void pick_tile_of_many(const AttWork& w, uint32_t index, uint32_t* sums,
                                                  AttLoad* loads, TilePick* pick) {
  const bool few = w.shared && AttLoad::of_call<kTileThreads / 32>(w, loads).splits();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t per = (w.kv.batch + kTileThreads - 1) / kTileThreads;
  const uint32_t b0 = min(w.kv.batch, tid * per), b1 = min(w.kv.batch, b0 + per);
  int first = 0, count = 0, len = 0;
  auto tiles = [&](uint32_t b) {
    w.kv.rows(b, w.tokens, &first, &count);
    len = w.kv.len(b);
    return tile_count(w, count, few);
  };
  uint32_t n = 0;
  for (uint32_t b = b0; b < b1; ++b) n += tiles(b);
  uint32_t inc = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sums[warp] = inc;
  if (tid == 0) pick->seq = 0xffffffffu;
  __syncthreads();
  uint32_t at = inc - n;
  for (int i = 0; i < warp; ++i) at += sums[i];
  if (index >= at && index < at + n) {
    uint32_t b = b0, last;
    for (; index >= at + (last = tiles(b)); ++b) at += last;
    *pick = {b, last - 1 - (index - at), first, count, len};
  }
  __syncthreads();
}

// Pages as heads: how many head strides a page stride is; 0 where the two do
// not make one dimension, or where a dimension that is walked has a stride of 0
// (a broadcast view; a tensor map is not made of one). The split kernel then
// takes the call.
inline uint64_t tile_heads_per_page(const PagedView& kv) {
  if (kv.pages == 0 || kv.st <= 0 || (kv.n_kv > 1 && kv.sh <= 0) || (kv.pages > 1 && kv.sp <= 0))
    return 0;
  if (kv.n_kv == 1 || kv.pages == 1) return kv.n_kv;
  if (kv.sp % kv.sh != 0 || kv.sp / kv.sh < static_cast<int64_t>(kv.n_kv)) return 0;
  const uint64_t per = static_cast<uint64_t>(kv.sp / kv.sh);
  return per * (kv.pages + 1) < (1ull << 31) ? per : 0;
}

template <int DT, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attention_tile_kernel(const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v,
                          const __grid_constant__ TileArgs a) {
  using L = TileLayout<D>;
  constexpr int NS = L::kStages;
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* empty = full + NS;
  uint64_t* q_full = empty + NS;
  uint64_t* s_full = q_full + 1;   // [2]: the slot holds the scores of half h
  uint64_t* s_free = s_full + 2;   // they are in registers
  uint64_t* p_full = s_free + 1;   // [2]: the weights are written, O is rescaled
  uint64_t* pv_done = p_full + 2;  // [2]: PV_h(j) is complete
  uint64_t* drain = pv_done + 2;  // [2]: of the issuers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  __shared__ uint32_t s_bad[8], s_sum[kTileThreads / 32];
  __shared__ TilePick s_tile;
  const AttWork& w = a.w;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], kTileLoaders);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 512);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(s_free, 8);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbarrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 16) tmem_alloc(tmem_slot, kTmemCols);
  pdl_wait();
  pdl_launch_dependents();
  // ---- which tile: those with the most key blocks first, the kv heads of one
  // side by side
  const uint32_t index = blockIdx.x / w.kv.n_kv, hk = blockIdx.x - index * w.kv.n_kv;
  TilePick t;
  if (w.kv.batch <= 32) {
    t = pick_tile(w, index);  // by every warp for itself
  } else {
    pick_tile_of_many(w, index, s_sum, reinterpret_cast<AttLoad*>(smem), &s_tile);
    t = s_tile;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (t.seq == 0xffffffffu) {  // the grid is sized for the most tiles there can be
    if (warp == 16) tmem_dealloc(*tmem_slot, kTmemCols);
    return;
  }

  // ---- the tile's rows and key blocks
  const uint32_t b = t.seq;
  const int first = t.first, count = t.count, len = t.len;
  const uint32_t rows = static_cast<uint32_t>(count) * w.group;
  const uint32_t p0 = t.tile * w.row_tile, p1 = min(p0 + w.row_tile, rows);
  const bool two = p0 + 128 < p1;
  const int shift = len - count;  // position of the first new token
  const int pos_lo = shift + static_cast<int>(w.by_group.div(p0));
  const int pos_hi = shift + static_cast<int>(w.by_group.div(p1 - 1));
  const int start = w.window_start(pos_lo);
  // past the table's end there is nothing: no blocks, and keys of the last one
  // that lie there count as a page that is missing
  const int last = min(pos_hi, w.kv.cap() - 1);
  const int head = (min(min(w.sinks, start), last + 1) + kTileKeys - 1) / kTileKeys;  // blocks that hold sinks
  const int main0 = max(start / kTileKeys, head);
  const int nb = last < 0 ? 0 : head + max(0, last / kTileKeys - main0 + 1);
  auto block_key = [&](int j) { return (j < head ? j : main0 + j - head) * kTileKeys; };

  const uint32_t tmem = *tmem_slot;
  const uint32_t sm = smem_u32(smem);

  if (warp < 16) {
    // ---------------------------------------------------------- softmax
    const int half = warp >> 3;
    // both halves' rows of q into shared memory, K-major with 128-byte swizzle
    constexpr int CPR = D / 8;
#pragma unroll 8
    for (uint32_t r = tid / CPR; r < (two ? 256u : 128u); r += 512 / CPR) {
      const uint32_t c = tid % CPR, p = p0 + r, tok = w.by_group.div(p);
      cp_async_16(sm + (r >> 7) * L::kHalf + (c >> 3) * L::kBlk + (r & 127) * 128 +
                      (((c & 7) ^ (r & 7)) << 4),
                  p < rows ? a.q + (first + tok) * a.ld_q +
                                 static_cast<int64_t>(hk * w.group + p - tok * w.group) * (2 * D) +
                                 16 * c
                           : a.q,
                  p < rows ? 16 : 0);
    }
    cp_async_commit();
    cp_async_wait<0>();
    fence_proxy_async_smem();
    mbar_arrive(q_full);

    if (half == 0 || two) {
      // this thread's rows r0 and r0 + 8 of the half, columns 8 j + 2 (lane % 4), + 1
      const int t4 = lane & 3, r0 = 32 * (warp & 3) + 16 * ((warp >> 2) & 1) + (lane >> 2);
      const uint32_t lanes = static_cast<uint32_t>(r0 & ~15) << 16;
      const uint32_t ts = tmem + lanes, tp = tmem + lanes + 128 + 64 * half;
      const uint32_t to = tmem + lanes + 256 + 128 * half;
      const float sl = a.scale_log2, slack = kTileSlack / sl;
      const uint64_t sl2 = f2_pack(sl, sl);
      bool have[2];
      int pos[2];
      float m[2], l[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t p = p0 + 128 * half + r0 + 8 * i;
        have[i] = p < rows;
        pos[i] = shift + static_cast<int>(w.by_group.div(have[i] ? p : 0u));
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      bool ok = true;
      for (int j = 0; j < nb; ++j) {
        ok = mbar_wait_prompt(&s_full[half], j & 1);
        ok = __all_sync(0xffffffffu, ok);  // tcgen05.ld / st are warp-collective
        if (!ok) break;
        tc_fence_after();
        float s[2][32];
        tmem_ld_16x256b_x8_nowait(ts, s[0]);
        tmem_ld_16x256b_x8_nowait(ts + 64, s[1]);
        const int key0 = block_key(j);
        const uint32_t bad = s_bad[j & 7];
        bool open = bad == 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          open = open && (!have[i] || (key0 + kTileKeys - 1 <= pos[i] &&
                                       (w.window == 0 || key0 > pos[i] - w.window ||
                                        key0 + kTileKeys - 1 < w.sinks)));
        const bool cut = !__all_sync(0xffffffffu, open);
        tmem_wait_ld(s[0]);
        tmem_wait_ld(s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if (cut) {
          // a row's visible keys as bits: up to its position, and in the window
          // or among the sinks. (hi - window may wrap where hi <= 0: nothing is
          // seen then, whatever lo is.)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int hi = pos[i] - key0 + 1;
            const int lo = w.window > 0 ? static_cast<int>(static_cast<uint32_t>(hi) - w.window) : 0;
            const int si = w.sinks - key0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t see =
                  low_bits(hi - 32 * c) & (~low_bits(lo - 32 * c) | low_bits(si - 32 * c));
              if (bad != 0) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (bad >> (4 * c + k) & 1) see &= ~(0xffu << 8 * k);
              }
              see >>= 2 * t4;
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& v = s[c >> 1][16 * (c & 1) + 4 * k + 2 * i + e];
                  v = see >> (8 * k + e) & 1 ? v : -INFINITY;
                }
            }
          }
        }
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float t[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            t[c] = fmaxf(s[c][2 * i], s[c][2 * i + 1]);
#pragma unroll
            for (int k = 1; k < 8; ++k) t[c] = max3(t[c], s[c][4 * k + 2 * i], s[c][4 * k + 2 * i + 1]);
          }
          top[i] = fmaxf(t[0], t[1]);
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + slack || top[1] > m[1] + slack)) {
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float mn = fmaxf(m[i], top[i]);
            f[i] = m[i] == -INFINITY ? 0.f : exp2_approx((m[i] - mn) * sl);
            l[i] *= f[i];
            m[i] = mn;
          }
          if (j > 0) {
            ok = mbar_wait_prompt(&pv_done[half], (j - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              float o[8];
              tmem_ld_16x256b_x2(to + 16 * c, o);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] *= f[k >> 1 & 1];
              tmem_st_16x256b_x2_nowait(to + 16 * c, o);
            }
          }
        }
        uint64_t nb2[2], sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float base = m[i] == -INFINITY ? 0.f : m[i] * sl;
          nb2[i] = f2_pack(-base, -base);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {  // repetition k / 2, row k % 2
            const uint64_t x2 =
                f2_fma(f2_pack(s[c][2 * k], s[c][2 * k + 1]), sl2, nb2[k & 1]);
            float x, y;
            f2_unpack(x2, x, y);
            x = exp2_approx(x);
            y = exp2_approx(y);
            sum[k & 1] = f2_add(sum[k & 1], f2_pack(x, y));
            pk[k] = pack2<DT>(x, y);
          }
          if (c == 0 && j > 0) {  // PV(j - 1) has read the weights' place
            ok = mbar_wait_prompt(&pv_done[half], (j - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
          }
          tmem_st_16x128b_x8_nowait(tp + 32 * c, pk);
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x, y;
          f2_unpack(sum[i], x, y);
          l[i] += x + y;
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[half]);
      }
      if (ok && nb > 0) {
        ok = mbar_wait_prompt(&pv_done[half], (nb - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok) {
        char* dst[2];
        float inv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 1; d < 4; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
          // without a maximum the sum is 0, no key seen, or NaN, a query that is
          // not finite: the row's output too
          inv[i] = m[i] != -INFINITY ? 1.f / l[i] : l[i];
          const uint32_t p = p0 + 128 * half + r0 + 8 * i, tok = w.by_group.div(have[i] ? p : 0u);
          dst[i] = a.out + (first + tok) * a.ld_o +
                   static_cast<int64_t>(hk * w.group + p - tok * w.group) * (2 * D);
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          float o[32];
          if (nb > 0) {
            tmem_ld_16x256b_x8_nowait(to + 64 * c, o);
            tmem_wait_ld(o);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // the four threads of a row trade their pieces of four repetitions,
            // so that each stores 16 bytes: thread t4 those of repetition 4 q + t4
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float* e = o + 4 * (4 * q + k) + 2 * i;
                v[k] = inv[i] != 0.f ? pack2<DT>(e[0] * inv[i], e[1] * inv[i]) : 0u;
              }
              quad_transpose(v, t4);
              if (have[i])
                *reinterpret_cast<uint4*>(dst[i] + 128 * c + 64 * q + 16 * t4) =
                    make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
      }
    }
  } else if (warp == 16) {
    // ------------------------------------------ issuer of the score products
    // (the whole warp runs the loop, one thread issues)
    const bool leader = elect_one();
    const uint32_t id_s = tw_idesc(DT == kBF16, kTileKeys) | a.negate;
    const uint64_t qd = umma_desc_sw128(sm, 16, 1024);
    const uint64_t kd = umma_desc_sw128(sm + L::kOffKV, 16, L::kGroup);
    const int halves = two ? 2 : 1;
    uint32_t scores = 0;  // score products issued; each needs the slot of the one before
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && mbar_wait_prompt(bar, parity);
      ok = __all_sync(0xffffffffu, ok);
    };
    if (nb > 0) wait(q_full, 0);
    for (int j = 0; j < nb && ok; ++j) {
      const uint32_t st = tile_stage_k(j), slot = st % NS;
      wait(&full[slot], st / NS & 1);
      for (int h = 0; h < halves; ++h) {
        if (scores > 0) wait(s_free, (scores - 1) & 1);
        if (!ok) break;
        ++scores;
        tc_fence_after();
        if (leader) {
          const uint64_t q = qd + h * (L::kHalf >> 4), k = kd + slot * (L::kHalf >> 4);
#pragma unroll
          for (int x = 0; x < D / 16; ++x)  // descriptors count 16-byte units
            umma_f16(tmem, q + 2 * (x & 3) + (x >> 2) * (L::kBlk >> 4),
                     k + 2 * (x & 3) + (x >> 2) * (1024 >> 4), id_s, x > 0);
          umma_commit(&s_full[h]);
          if (h + 1 == halves) umma_commit(&empty[slot]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (leader) umma_commit(&drain[0]);
      __syncwarp();
      mbar_wait_bounded(&drain[0], 0);
    }
  } else if (warp == 17) {
    // ----------------------------------------- issuer of the second products
    const bool leader = elect_one();
    constexpr uint32_t id_o = umma_idesc_f16(DT == kBF16, 128, D);
    const uint64_t vd = umma_desc_sw128(sm + L::kOffKV, 1024, L::kGroup);
    const int halves = two ? 2 : 1;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && mbar_wait_prompt(bar, parity);
      ok = __all_sync(0xffffffffu, ok);
    };
    for (int j = 0; j < nb && ok; ++j) {
      const uint32_t st = tile_stage_v(j, nb), slot = st % NS;
      wait(&full[slot], st / NS & 1);
      for (int h = 0; h < halves; ++h) {
        wait(&p_full[h], j & 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t o = tmem + 256 + 128 * h, p = tmem + 128 + 64 * h;
          const uint64_t v = vd + slot * (L::kHalf >> 4);
#pragma unroll
          for (int x = 0; x < kTileKeys / 16; ++x)
            umma_f16_tmem_a(o, p + 8 * x, v + x * (2 * L::kGroup >> 4), id_o, j > 0 || x > 0);
          umma_commit(&pv_done[h]);
          if (h + 1 == halves) umma_commit(&empty[slot]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (leader) umma_commit(&drain[1]);
      __syncwarp();
      mbar_wait_bounded(&drain[1], 0);
    }
  } else {
    // ------------------------------------------------- K / V producers
    const int loader = warp - 18;
    const uint32_t box_keys = a.box, boxes = kTileKeys / box_keys;  // of a block
    const uint32_t box_bytes = box_keys * 2 * D;
    int slot = 0, issued = 0;
    uint32_t par = 1;  // parity of the slot's last release (a fresh barrier: done)
    bool ok = true;
    const int seen = min(len, pos_hi + 1), sinks = min(w.sinks, start);
    const int32_t* table = w.kv.table + b * w.kv.ld_table;
    // lane i < boxes looks up box i of a block: its page (one block ahead of
    // its use), and where the sequence ends
    struct Box {
      int key, page, in_page;
      bool need;
      uint32_t bad, cuts;
    };
    auto fetch = [&](int j) {
      Box x;
      x.key = (j < head ? j : main0 + j - head) * kTileKeys + static_cast<int>(lane * box_keys);
      x.need = j < nb && lane < boxes && x.key < seen &&
               (x.key + static_cast<int>(box_keys) > start || x.key < sinks);
      const uint32_t pg = x.need ? w.kv.page.div(x.key) : 0u;
      x.in_page = x.need ? x.key - static_cast<int>(pg * w.kv.page.d) : 0;
      x.page = x.need && pg < w.kv.width ? table[pg] : -1;
      return x;
    };
    auto find = [&](Box& x) {
      const bool there = static_cast<uint32_t>(x.page) < w.kv.pages;
      const uint32_t gone = __ballot_sync(0xffffffffu, x.need && !there);
      x.bad = 0;
      if (gone != 0) {
        if (lane == 0) atomicOr(&g_cawq_device_error, kErrCache);
        // the same by groups of 8 keys
        x.bad = __ballot_sync(0xffffffffu, lane < 16 && (gone >> (8 * lane / box_keys) & 1));
      }
      x.cuts = __ballot_sync(0xffffffffu, there && x.key + static_cast<int>(box_keys) > len);
      // past the last page: the box is outside the tensor and arrives as zeros
      if (!there) x.page = static_cast<int>(w.kv.pages);
    };
    auto load = [&](const Box& x, bool values) {
      ok = ok && mbar_wait_prompt(&empty[slot], par);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      const uint32_t dst = L::kOffKV + slot * L::kHalf;
      const uint32_t cuts = values ? x.cuts : 0u;
      if (cuts != 0 && loader == 0) {
        // the values of the last page, with zeros past the sequence's end
        const int from = __ffs(cuts) - 1;
        const int pg = __shfl_sync(0xffffffffu, x.page, from);
        const int ip = __shfl_sync(0xffffffffu, x.in_page, from);
        const int left = len - __shfl_sync(0xffffffffu, x.key, from);
        const char* src = w.kv.v + pg * w.kv.sp + hk * w.kv.sh + ip * w.kv.st;
        for (uint32_t i = lane; i < box_keys * (D / 8); i += 32) {
          const uint32_t r = i / (D / 8), c = i % (D / 8), rr = from * box_keys + r;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (static_cast<int>(r) < left)
            v = *reinterpret_cast<const uint4*>(src + r * w.kv.st + 16 * c);
          *reinterpret_cast<uint4*>(smem + dst + (rr >> 3) * L::kGroup + (c >> 3) * 1024 +
                                    (rr & 7) * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v;
        }
        fence_proxy_async_smem();
        __syncwarp();  // lane 0's arrival speaks for all lanes' writes
      }
      // the boxes are dealt out to the loaders' lanes
      const uint32_t box = lane * kTileLoaders + loader;
      const int page = __shfl_sync(0xffffffffu, x.page, box & 31);
      const int in_page = __shfl_sync(0xffffffffu, x.in_page, box & 31);
      const bool mine = box < boxes && !(cuts >> box & 1);
      const uint32_t count = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_arrive_expect_tx(&full[slot], count * box_bytes);
      __syncwarp();
      if (mine)
        tma_load_5d(sm + dst + box * box_bytes, values ? &tm_v : &tm_k, 0, 0, 0, in_page / 8,
                    static_cast<int>(page * a.heads_per_page + static_cast<int>(hk)), &full[slot]);
      __syncwarp();
      ++issued;
      if (++slot == NS) {
        slot = 0;
        par ^= 1u;
      }
    };
    if (nb > 0) {
      Box now = fetch(0), after = fetch(1);
      find(now);
      if (loader == 0 && lane == 0) s_bad[0] = now.bad;
      load(now, false);
      for (int j = 0; j < nb && ok; ++j) {
        Box next = after;
        if (j + 1 < nb) {
          after = fetch(j + 2);
          find(next);
          if (loader == 0 && lane == 0) s_bad[(j + 1) & 7] = next.bad;
          load(next, false);
        }
        if (ok) load(now, true);
        now = next;
      }
    }
    if (!ok) {  // copies in flight end before the CTA does
      for (int i = max(0, issued - NS); i < issued; ++i)
        mbar_wait_bounded(&full[i % NS], (i / NS) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// The cache's keys or values as a 5-D tensor: 64 elements, 8 slots, column
// blocks, groups of 8 slots, heads (those of a page follow those of the page
// before). A box then lands group by group, column block by column block: one
// copy per page brings every column. (TMA takes 60 cycles or more for a box
// however small: with a box per column block, pages of 16 made the loads the
// bound, 1400 cycles a stage.) False if the strides do not fit.
inline bool encode_cache(CUtensorMap* map, int dtype, const void* base, const PagedView& kv,
                         uint32_t d, uint32_t box) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  // an extent of 1 never uses its stride, which may then be anything
  const uint64_t sh = kv.n_kv > 1 || kv.pages > 1 ? kv.n_kv > 1 ? kv.sh : kv.sp : 2 * d;
  const uint64_t per = tile_heads_per_page(kv);
  const uint64_t dims[5] = {64, 8, d / 64, kv.page.d / 8, (kv.pages - 1) * per + kv.n_kv};
  const uint64_t strides[4] = {static_cast<uint64_t>(kv.st), 128, 8 * static_cast<uint64_t>(kv.st), sh};
  const uint32_t bx[5] = {64, 8, d / 64, box / 8, 1}, es[5] = {1, 1, 1, 1, 1};
  return fn(map, dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            5, const_cast<void*>(base), dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == 0;
}

template <int DT, int D>
cudaError_t launch_attention_tile_t(const AttentionProblem& p, const PagedView& kv, bool shared) {
  static uint64_t done = 0;
  auto kern = attention_tile_kernel<DT, D>;
  cudaError_t e = allow_smem(kern, TileLayout<D>::kSmem, p.device, &done);
  if (e != cudaSuccess) return e;
  TileArgs a;
  a.q = static_cast<const char*>(p.q);
  a.out = static_cast<char*>(p.out);
  a.w = att_work(p, kv, 0, shared);
  a.ld_q = static_cast<int64_t>(p.ld_q) * 2;
  a.ld_o = static_cast<int64_t>(p.ld_out) * 2;
  // scores of a scale of 0 are all equal: so they are at 1e-30
  a.scale_log2 = std::max(std::abs(p.scale) * kLog2e, 1e-30f);
  a.negate = p.scale < 0 ? 1u << 13 : 0u;
  a.box = 8;
  while (a.box < kTileKeys && kv.page.d % (2 * a.box) == 0) a.box *= 2;
  a.heads_per_page = static_cast<int64_t>(tile_heads_per_page(kv));
  CUtensorMap mk, mv;
  if (!encode_cache(&mk, DT, kv.k, kv, D, a.box) || !encode_cache(&mv, DT, kv.v, kv, D, a.box))
    return cudaErrorInvalidValue;
  // Tiles of one half where the CTAs of two would leave half the SMs idle, since
  // a block of keys takes less time with one: 77 tokens, 14 / 2 heads, D = 64,
  // 6.9 against 7.8 us, 500 tokens 10.6 against 13.0; 64 to 500 new tokens after
  // 2000, 32 / 8 heads, D = 128, 27 to 31.5 against 35 to 40.
  uint64_t tiles = 0;
  for (a.w.row_tile = kTileRows;; a.w.row_tile /= 2) {
    tiles = p.tokens * a.w.group / a.w.row_tile + std::min<uint64_t>(kv.batch, p.tokens);
    if (a.w.row_tile < kTileRows || 2 * tiles * kv.n_kv > static_cast<uint64_t>(p.sm_count)) break;
  }
  void* args[] = {&mk, &mv, &a};
  return launch_pdl(kern, dim3(static_cast<uint32_t>(tiles * kv.n_kv)), kTileThreads,
                    TileLayout<D>::kSmem, p.stream, args);
}

cudaError_t launch_attention_tile(const AttentionProblem& p, const PagedView& kv, bool shared) {
  if (p.dtype == kF16)
    return p.d == 64 ? launch_attention_tile_t<kF16, 64>(p, kv, shared)
                     : launch_attention_tile_t<kF16, 128>(p, kv, shared);
  return p.d == 64 ? launch_attention_tile_t<kBF16, 64>(p, kv, shared)
                   : launch_attention_tile_t<kBF16, 128>(p, kv, shared);
}

}  // namespace cawq
