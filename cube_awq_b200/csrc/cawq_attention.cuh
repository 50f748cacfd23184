// cawq_attention.cuh — attention of few query rows over a paged cache, split
// over the cache's length (sm_100a): one new token per sequence, or short runs
// of them.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// over the visible positions, m their running maximum. Two parts with their
// own maxima join exactly: with M = max(m1, m2), sum = 2^(m1 - M) sum1 +
// 2^(m2 - M) sum2, the same for the outputs.
//
// Bound by the cache's bytes (one sequence of 131072 tokens, 64 / 8 heads, bf16:
// 537 MB in 88-91 us, 5.9-6.1 TB/s) and, below some 100 MB, by what a launch costs at
// its ends, 8 us with the join (64 sequences of 1 to 8000 tokens, 28 / 4 heads:
// 133 MB in 33 us): every visible key and value is read once per tile of query
// rows that shares its kv head. A row tile is NR = 8 or 16 rows
// of one (sequence, kv head): the G = n_q / n_kv query heads of its tokens,
// token by token. All (row tile, 64-key tile) units of the batch, sequences of
// any length, form one list that is dealt out evenly to a grid of two CTAs per
// SM, so a batch of ragged lengths and one long sequence fill the GPU alike;
// the lengths are read on the device. A CTA's share may begin or end inside a
// row tile's keys: it then leaves its part (m, sum, outputs, fp32) in the
// workspace and a second small kernel joins the parts in order (no atomics:
// the same bits every time). Where the keys of each row tile are few, by the
// table's width, the dealing out costs more than it evens out, and a cluster of
// CTAs or a single warp takes the row tile instead (att_cluster, att_each).
//
// A CTA is four warps that never wait for one another inside a row tile: warp
// w takes keys 16 w .. 16 w + 15 of each 64-key tile and streams them through
// a ring of its own in shared memory (cp.async, 16 bytes a lane, rows swizzled
// so that ldmatrix reads without bank conflicts; a masked row is filled with
// zeros and never read). The stream runs on across row tiles. With mma.sync
// m16n8k16 the keys are the MMA's rows: S^T = K Q^T needs only N = 8 columns
// for 8 query rows; the weights, rounded to the operand type, which is what the
// instruction takes, turn in registers (movmatrix) into the B operand of O^T +=
// V^T P^T. The sums take them unrounded. Against 64 bits the output's error is
// 2.0e-3 in bf16, 2.2e-4 in f16, where weights of 32 bits leave 1.6e-3 and 2.1e-4
// (relative, 131072 and 1000 tokens).
#pragma once

#include "cawq_norm.cuh"
#include "cawq_paged.cuh"

namespace cawq {

constexpr int kAttWarps = 4;
constexpr int kAttKeys = 16 * kAttWarps;  // keys of a unit
constexpr int kAttStages = 3;
// Units that a row tile counts for beside its key tiles: beginning and ending
// one (rows of q, the join of the warps, the output) takes a CTA about as long
// as streaming two tiles. Without it a batch of many short sequences and a few
// long ones left the CTAs with the short ones last (64 sequences of 1 to 8000
// tokens, 28 / 4 heads: 62 us).
constexpr uint32_t kAttRowCost = 2;
// A sequence of at most so many query rows (of a kv head) is for the split
// kernel where a call's keys are worth splitting (AttLoad).
constexpr uint32_t kAttFewRows = 128;
constexpr uint32_t kAttMaxCluster = 16;  // most CTAs of a cluster that shares a row tile
constexpr uint32_t kAttClusterTiles = 8;  // most key tiles a CTA of it may get
// Most keys of a row tile that one warp takes: of those in two waves of CTAs, of others.
constexpr uint32_t kAttEachFew = 128, kAttEachKeys = 256;
constexpr int kAttMaxCtas = 320;  // most CTAs of a launch (two per SM)

template <int D>
struct AttLayout {
  static constexpr int kRow = 2 * D;            // bytes of a key
  static constexpr int kStage = 2 * 16 * kRow;  // keys and values of 16 positions
  static constexpr int kRing = kAttWarps * kAttStages * kStage;
  static constexpr int kPad = D + 4;  // floats of a merge row: 2 kPad = 8 (mod 32) banks
  static constexpr int kMerge = kAttWarps * 8 * kPad * 4;
  static constexpr int kSmem = kRing + kMerge;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes global -> shared; zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 8x8 b16 matrix transposed across the warp: lane (g, t) gives elements
// (g, 2t), (g, 2t + 1) and receives (2t, g), (2t + 1, g).
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    r = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
}

// What a launch works on; both kernels walk the same list of units.
struct AttWork {
  PagedView kv;
  uint32_t tokens, group, row_tile;  // group = n_q / n_kv, row_tile = NR
  FastDiv by_group;
  int window, sinks;
  bool shared;  // both kernels run: the tile kernel takes what the split kernel leaves

  // Sequence b: its rows, its keys in order of position without the hidden
  // ones between the sinks and the window of its first new token, and its
  // units: kv heads x row tiles x (kAttRowCost, then 64-key tiles). A sequence with new tokens
  // and no keys has one tile per row tile all the same: its rows are zeros.
  struct Seq {
    int first, count, len, start, head, keys;
    uint32_t tiles, row_tiles;
    __device__ __forceinline__ int key(int c) const { return c < head ? c : c - head + start; }
  };
  // the first position in the window of position pos (which may lie so far
  // below zero that pos - window passes 32 bits)
  __device__ __forceinline__ int window_start(int pos) const {
    return window > 0 && pos >= window ? pos - window + 1 : 0;
  }
  __device__ __forceinline__ Seq seq(uint32_t b) const {
    Seq s;
    kv.rows(b, tokens, &s.first, &s.count);
    s.len = kv.len(b);
    const int pos = s.len - s.count;  // of the first new token
    s.start = window_start(pos);
    const int end = min(s.len, kv.cap());
    s.head = min(min(sinks, s.start), end);
    s.keys = max(0, end - s.start) + s.head;
    s.row_tiles = (static_cast<uint32_t>(s.count) * group + row_tile - 1) / row_tile;
    s.tiles = s.count > 0 && (!shared || s.count * group <= kAttFewRows)
                  ? max(1, (s.keys + kAttKeys - 1) / kAttKeys)
                  : 0u;
    return s;
  }
  __device__ __forceinline__ uint64_t units(const Seq& s) const {
    return s.tiles ? static_cast<uint64_t>(s.tiles + kAttRowCost) * s.row_tiles * kv.n_kv : 0;
  }
};

// Whether a call's sequences of few rows go to the split kernel, by what all its
// sequences need. A tile reads a key in 9.4 ns and the GPU streams 11.8 keys a
// ns, kPole in that time; the split kernel reads a sequence's keys once per row
// tile of 16, but no CTA waits for the longest. So it gains where the longest
// sequence of few rows, less what its two launches cost, has more keys than all
// row tiles together have per kPole. us split against tiles (bf16, 8 kv heads,
// all of 1000 / 4000 / 16000 tokens), D = 128: 1 sequence of 16 rows 14 / 17 / 27
// against 15 / 42 / 149, of 128 rows 20 / 35 / 93 against 16 / 44 / 151; 8 of 16
// rows 21 / 39 / 100 against 22 / 52 / 160, of 64 rows 48 / 110 / 356 against
// 23 / 52 / 160; 32 of 16 rows and 1 to 8000 tokens 50 against 86. D = 64, whose
// blocks of keys take a tile as long and the split kernel not much less: 13 / 15 /
// 21 against 14 / 42 / 150, 17 / 30 / 77 against 15 / 43 / 152; 17 / 32 / 81
// against 20 / 50 / 160, 40 / 90 / 290 against 21 / 51 / 160; 41 against 85. The
// rule picks the faster of the two in all of them but 8 of 16 rows and 1000
// tokens, where it costs 3 us (D = 64) or nothing.
struct AttLoad {
  static constexpr uint32_t kPole = 111, kLaunch = 850;
  uint64_t keys;     // of the row tiles, or tiles, of all sequences
  uint32_t longest;  // of few rows
  __host__ __device__ __forceinline__ bool splits() const {
    return longest > kLaunch && static_cast<uint64_t>(longest - kLaunch) * kPole > keys;
  }
  // one sequence
  __device__ __forceinline__ static AttLoad of(const AttWork& w, int count, int len) {
    AttLoad a = {0, 0};
    if (count <= 0 || len <= 0) return a;
    const int64_t rows = static_cast<int64_t>(count) * w.group;
    int64_t n = min(len, w.kv.cap());
    if (w.window > 0) n = min(n, static_cast<int64_t>(w.window) + w.sinks + count);
    const bool few = rows <= kAttFewRows;
    if (few) a.longest = static_cast<uint32_t>(n);
    a.keys = static_cast<uint64_t>(n) * w.kv.n_kv * ((rows + (few ? 15 : 255)) / (few ? 16 : 256));
    return a;
  }
  __device__ __forceinline__ void add(const AttLoad& o) {
    keys += o.keys;
    longest = max(longest, o.longest);
  }
  __device__ __forceinline__ AttLoad of_warp() const {
    AttLoad a = *this;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      a.add({__shfl_xor_sync(0xffffffffu, a.keys, o), __shfl_xor_sync(0xffffffffu, a.longest, o)});
    return a;
  }
  // all sequences, by all of a CTA's warps; `part` holds one per warp
  template <int WARPS>
  __device__ __forceinline__ static AttLoad of_call(const AttWork& w, AttLoad* part) {
    AttLoad a = {0, 0};
    for (uint32_t b = threadIdx.x; b < w.kv.batch; b += 32 * WARPS) {
      int first, count;
      w.kv.rows(b, w.tokens, &first, &count);
      a.add(of(w, count, w.kv.len(b)));
    }
    a = a.of_warp();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    a = part[0];
    for (int i = 1; i < WARPS; ++i) a.add(part[i]);
    return a;
  }
};

// Exclusive prefix sums of the sequences' units, a run of sequences per thread
// of the CTA. att_find leaves the sequence that holds unit u and its
// first unit.
struct AttScan {
  static constexpr int W = kAttWarps;
  uint64_t part[32 * W];  // units before thread i's sequences
  uint64_t sums[W];       // of the warps
  uint64_t total, before;
  uint32_t seq;
  AttLoad loads[W];
};

__device__ __forceinline__ void att_scan(const AttWork& w, AttScan& sc) {
  constexpr int W = kAttWarps;
  const uint32_t per = (w.kv.batch + 32 * W - 1) / (32 * W);
  const uint32_t b0 = threadIdx.x * per, b1 = min(w.kv.batch, b0 + per);
  uint64_t n = 0;
  for (uint32_t b = b0; b < b1; ++b) n += w.units(w.seq(b));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sc.sums[warp] = inc;
  __syncthreads();
  uint64_t base = 0, all = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < warp) base += sc.sums[i];
    all += sc.sums[i];
  }
  sc.part[threadIdx.x] = base + inc - n;
  if (threadIdx.x == 0) sc.total = all;
  __syncthreads();
}

// After att_scan: the sequence that holds unit u (< total) and the units before it.
__device__ __forceinline__ void att_find(const AttWork& w, AttScan& sc, uint64_t u) {
  constexpr int W = kAttWarps;
  const uint32_t per = (w.kv.batch + 32 * W - 1) / (32 * W);
  const uint64_t lo = sc.part[threadIdx.x];
  const uint64_t hi = threadIdx.x + 1 < 32 * W ? sc.part[threadIdx.x + 1] : sc.total;
  if (u >= lo && u < hi) {
    uint64_t at = lo;
    uint32_t b = threadIdx.x * per;
    for (;; ++b) {
      const uint64_t n = w.units(w.seq(b));
      if (u < at + n) break;
      at += n;
    }
    sc.seq = b;
    sc.before = at;
  }
  __syncthreads();
}

// CTA c of n works on the key tiles among units [first(c), first(c + 1)); n is at most the number
// of units, so that no CTA between two of a row tile's is without a part.
__device__ __forceinline__ uint32_t att_ctas(uint64_t total, uint32_t launched) {
  return static_cast<uint32_t>(min(total, static_cast<uint64_t>(launched)));
}
__device__ __forceinline__ uint64_t att_first_unit(uint64_t total, uint32_t cta, uint32_t ctas) {
  return total * cta / ctas;
}

// The workspace begins with a note of each CTA on the row tile that it began
// and left to the next ones (parts = 0: none), for the joining kernel.
struct AttNote {
  uint32_t parts;  // parts of the row tile; that CTA's first
  uint32_t late;   // that CTA worked on another row tile before
  int first;       // row of q of the sequence's first token
  uint32_t hk, r0;
  int rows;
  uint32_t pad[2];
};
constexpr size_t kAttNotes = kAttMaxCtas * sizeof(AttNote);

// A part in the workspace: NR maxima, NR sums, NR x D outputs.
template <int D, int NR>
__device__ __forceinline__ float* att_slot(char* ws, uint32_t slot) {
  return reinterpret_cast<float*>(ws + kAttNotes) + static_cast<size_t>(slot) * NR * (D + 2);
}

// MULTI: sequences may have several new tokens, so rows of a tile see
// different keys. Without it every visible key is every row's.
// kAttCluster (one token per sequence): no dealing out; a cluster of CTAs per
// row tile splits its keys evenly and joins through distributed shared memory,
// in one launch without a workspace. kAttEach (the same): a warp per row tile,
// 16 keys at a time, the row tiles in turn; nothing to join at all.
enum AttMode { kAttDealt, kAttCluster, kAttEach };
template <int DT, int D, int NT, bool MULTI, AttMode MODE>
__global__ void __launch_bounds__(32 * kAttWarps, 2)
    attention_split_kernel(const char* q, char* out, const AttWork w, int64_t ld_q, int64_t ld_o,
                           float scale_log2, char* ws) {
  using T = typename DType<DT>::T;
  using L = AttLayout<D>;
  constexpr int NR = 8 * NT, KS = D / 16;
  constexpr bool CLUSTER = MODE == kAttCluster, EACH = MODE == kAttEach;
  extern __shared__ __align__(128) uint8_t smem[];
  AttScan& sc = *reinterpret_cast<AttScan*>(smem + L::kRing);  // read before the first merge
  // The warps' maxima and sums for their join stand in the merge rows' padding:
  // with 640 bytes more a CTA, two would not fit on an SM at D = 128 (250
  // sequences of 1000 tokens, 16 / 1 heads, dealt out: 63 against 45 us).
  float* merge = reinterpret_cast<float*>(smem + L::kRing);
  auto s_m = [&](int i, int r) -> float& { return merge[(8 * i + (r & 7)) * L::kPad + D + (r >> 3)]; };
  auto s_f = [&](int i, int r) -> float& { return merge[(8 * i + (r & 7)) * L::kPad + D + 2 + (r >> 3)]; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;

  pdl_wait();
  pdl_launch_dependents();  // after the wait: the joining kernel may read the lengths at once
  uint64_t total = 0, u1 = 0;
  uint32_t ctas = 0;
  AttNote* note = reinterpret_cast<AttNote*>(ws) + blockIdx.x;
  int64_t left;  // units not issued yet
  struct Cursor {
    uint32_t b, hr, tile;
    AttWork::Seq s;
    uint32_t item;  // EACH: the row tile, of all
  };
  Cursor in;
  // keys of a unit, and where the warp's own begin; EACH counts units of 16
  constexpr int UK = EACH ? 16 : kAttKeys;
  const int own_key = EACH ? 0 : 16 * warp;
  const uint32_t per_seq = w.kv.n_kv * ((w.group + NR - 1) / NR);  // row tiles, one token each
  auto place = [&](Cursor& c) {
    c.b = c.item / per_seq;
    c.hr = c.item - c.b * per_seq;
    c.tile = 0;
    c.s = w.seq(c.b);
    c.s.tiles = max(1, (c.s.keys + UK - 1) / UK);
  };
  uint32_t cluster = 1, rank = 0;
  if constexpr (EACH) {
    in.item = blockIdx.x * kAttWarps + warp;
    if (in.item >= w.kv.batch * per_seq) return;
    place(in);
    left = 1;
  } else if constexpr (CLUSTER) {
    cluster = cluster_nctarank();
    rank = cluster_ctarank();
    in.item = blockIdx.x / cluster;
    place(in);
    in.tile = in.s.tiles * rank / cluster;
    left = in.s.tiles * (rank + 1) / cluster - in.tile;
  } else {
    if (w.shared) {
      if (threadIdx.x == 0) note->parts = 0;
      if (!AttLoad::of_call<kAttWarps>(w, sc.loads).splits()) return;
    }
    att_scan(w, sc);
    total = sc.total;
    ctas = att_ctas(total, gridDim.x);
    if (threadIdx.x == 0) note->parts = 0;
    if (blockIdx.x >= ctas) return;
    const uint64_t u0 = att_first_unit(total, blockIdx.x, ctas);
    u1 = att_first_unit(total, blockIdx.x + 1, ctas);
    att_find(w, sc, u0);
    left = static_cast<int64_t>(u1 - u0);
    in.b = sc.seq;
    in.s = w.seq(in.b);
    const uint64_t rel = u0 - sc.before;
    in.hr = static_cast<uint32_t>(rel / (in.s.tiles + kAttRowCost));
    const uint32_t r = static_cast<uint32_t>(rel - static_cast<uint64_t>(in.hr) * (in.s.tiles + kAttRowCost));
    in.tile = r < kAttRowCost ? 0 : r - kAttRowCost;
    left -= r < kAttRowCost ? kAttRowCost - r : 0;
    __syncthreads();  // sc is read: the merge rows may be written
    if (left <= 0) return;  // nothing but the cost of a row tile that the next CTA begins
  }
  Cursor at = in;
  const int64_t left0 = left;
  // ---- the stream of 64-key tiles: a cursor that runs ahead of the work
  auto next_rows = [&](Cursor& c) {
    c.tile = 0;
    if (++c.hr < c.s.row_tiles * w.kv.n_kv) return;
    c.hr = 0;
    do {
      ++c.b;
      c.s = w.seq(c.b);
    } while (c.s.tiles == 0);
  };
  // one tile on, while there are units; false past the CTA's last tile
  auto advance = [&](Cursor& c, int64_t& units) -> bool {
    if constexpr (EACH) {
      if (++c.tile < c.s.tiles) return true;
      c.item += gridDim.x * kAttWarps;
      if (c.item >= w.kv.batch * per_seq) return false;
      place(c);
      return true;
    }
    --units;
    if (++c.tile < c.s.tiles) return units > 0;
    units -= kAttRowCost;
    if (units <= 0) return false;
    next_rows(c);
    return true;
  };
  // the lane's position (16 per warp) in the cache: byte offset, -1 if none
  auto lookup = [&](const Cursor& c) -> int64_t {
    const int i = static_cast<int>(c.tile * UK) + own_key + (lane & 15);
    if (i >= c.s.keys) return -1;
    return w.kv.offset(c.b, c.hr / c.s.row_tiles, static_cast<uint32_t>(c.s.key(i)));
  };
  const uint32_t ring = smem_u32(smem) + warp * (kAttStages * L::kStage);
  constexpr int CPR = L::kRow / 16;  // 16-byte chunks of a row
  constexpr int RPI = 32 / CPR;      // rows of one instruction
  auto issue = [&](int slot, int64_t off) {
    const uint32_t dst = ring + slot * L::kStage;
    const int col = lane % CPR;
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const int row = RPI * i + lane / CPR;
      const int64_t o = __shfl_sync(0xffffffffu, off, row);
      const uint32_t d = dst + row * L::kRow + ((col ^ (row & 7)) << 4);
      const int64_t a = o < 0 ? 0 : o + 16 * col;
      cp_async_16(d, w.kv.k + a, o < 0 ? 0 : 16);
      cp_async_16(d + 16 * L::kRow, w.kv.v + a, o < 0 ? 0 : 16);
    }
  };

  int64_t todo = left;  // units not worked off yet
  bool more = left > 0;  // `in` stands on a tile of this CTA's
  uint32_t masks[kAttStages];
  int64_t off = lookup(in);
  auto refill = [&](int slot) -> uint32_t {
    uint32_t mask = 0;
    if (more) {
      mask = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
      issue(slot, off);
      more = advance(in, left);
      if (more) off = lookup(in);
    }
    cp_async_commit();
    return mask;
  };
#pragma unroll
  for (int i = 0; i < kAttStages - 1; ++i) masks[i] = refill(i);
  masks[kAttStages - 1] = 0;

  // ---- the rows of the current row tile
  uint32_t qf[NT][KS][2];
  float m[NT][2], l[NT][2], o[NT][KS][4];
  int prow[NT][2];  // MULTI: position of the lane's rows, -1 for none
  auto load_rows = [&](const Cursor& c) {
    const uint32_t hk = c.hr / c.s.row_tiles;
    const uint32_t r0 = (c.hr - hk * c.s.row_tiles) * NR;
    const uint32_t rows = static_cast<uint32_t>(c.s.count) * w.group;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const uint32_t r = r0 + 8 * x + g;
      const uint32_t tok = w.by_group.div(r);
      const bool have = r < rows;
      const T* src = reinterpret_cast<const T*>(
          q + (have ? (c.s.first + tok) * ld_q +
                          static_cast<int64_t>(hk * w.group + r - tok * w.group) * (2 * D)
                    : 0));
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[x][s][0] = have ? *reinterpret_cast<const uint32_t*>(src + 16 * s + 2 * t4) : 0u;
        qf[x][s][1] = have ? *reinterpret_cast<const uint32_t*>(src + 16 * s + 8 + 2 * t4) : 0u;
      }
      if constexpr (MULTI) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t rr = r0 + 8 * x + 2 * t4 + k;
          prow[x][k] = rr < rows ? c.s.len - c.s.count + static_cast<int>(w.by_group.div(rr)) : -1;
        }
      }
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[x][s][c] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[x][c] = -INFINITY;
        l[x][c] = 0.f;
      }
    }
  };
  load_rows(at);
  clear();
  uint32_t tile0 = at.tile;

  // ldmatrix addresses: lane L gives row L & 7 of matrix L >> 3
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t k_row = ((mi & 1) * 8 + mr) * L::kRow, v_row = ((mi >> 1) * 8 + mr) * L::kRow;

  int slot = 0;
  for (bool first_rows = true; !CLUSTER || todo > 0;) {
    cp_async_wait<kAttStages - 2>();
    __syncwarp();
    {
      // refill the slot that the previous tile left
      const int fill = slot == 0 ? kAttStages - 1 : slot - 1;
      const uint32_t mk = refill(fill);
#pragma unroll
      for (int i = 0; i < kAttStages; ++i)
        if (i == fill) masks[i] = mk;
    }
    uint32_t mask = masks[0];
#pragma unroll
    for (int i = 1; i < kAttStages; ++i)
      if (i == slot) mask = masks[i];
    const uint32_t kb = ring + slot * L::kStage, vb = kb + 16 * L::kRow;

    // S^T = K Q^T: lane holds keys g and g + 8 of rows 2 t4, 2 t4 + 1
    float s[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[x][c] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4(kb + k_row + (((2 * i + (mi >> 1)) ^ mr) << 4), a0, a1, a2, a3);
#pragma unroll
      for (int x = 0; x < NT; ++x)
        mma_16816<DT == kBF16>(s[x], a0, a1, a2, a3, qf[x][i][0], qf[x][i][1]);
    }
    const bool in0 = (mask >> g) & 1, in1 = (mask >> (g + 8)) & 1;
    uint32_t pb[NT][2];
    bool moved = false;
    float corr[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        bool see = c < 2 ? in0 : in1;
        if constexpr (MULTI) {
          const int key = at.s.key(static_cast<int>(at.tile * UK) + own_key + g + (c < 2 ? 0 : 8));
          const int p = prow[x][c & 1];
          see = see && key <= p && (w.window == 0 || p - key < w.window || key < w.sinks);
        }
        v[c] = see ? s[x][c] * scale_log2 : -INFINITY;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = fmaxf(v[c], v[c + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float mn = fmaxf(m[x][c], top);
        const float base = mn == -INFINITY ? 0.f : mn;
        corr[x][c] = exp2_approx(m[x][c] - base);
        moved |= mn != m[x][c];
        m[x][c] = mn;
        v[c] = exp2_approx(v[c] - base);
        v[c + 2] = exp2_approx(v[c + 2] - base);
        l[x][c] = l[x][c] * corr[x][c] + v[c] + v[c + 2];
      }
      // weights of the second product in the operand type, keys along k
      pb[x][0] = movmatrix_trans(pack2<DT>(v[0], v[1]));
      pb[x][1] = movmatrix_trans(pack2<DT>(v[2], v[3]));
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[x][i][c] *= corr[x][c & 1];
    }
    // O^T += V^T P^T: lane holds dimensions 16 i + g, + 8 of its two rows
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4_trans(vb + v_row + (((2 * i + (mi & 1)) ^ mr) << 4), a0, a1, a2, a3);
#pragma unroll
      for (int x = 0; x < NT; ++x) mma_16816<DT == kBF16>(o[x][i], a0, a1, a2, a3, pb[x][0], pb[x][1]);
    }
    __syncwarp();
    if (++slot == kAttStages) slot = 0;

    const Cursor done = at;
    const bool go_on = advance(at, todo);
    if (go_on && at.tile != 0) continue;
    // ---- the row tile's keys in this CTA end here: join the four warps
    const bool whole = CLUSTER ? cluster == 1 : tile0 == 0 && done.tile + 1 == done.s.tiles;
    if (go_on) load_rows(at);  // of the next one, while this one ends
    if constexpr (EACH) {
      const uint32_t hk = done.hr / done.s.row_tiles;
      const uint32_t r0 = (done.hr - hk * done.s.row_tiles) * NR;
      float* own = reinterpret_cast<float*>(smem + L::kRing) + warp * 8 * L::kPad;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], d);
          const float inv = l[x][c] != 0.f ? 1.f / l[x][c] : 0.f;
          float* dst = own + (2 * t4 + c) * L::kPad;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            dst[16 * i + g] = o[x][i][c] * inv;
            dst[16 * i + g + 8] = o[x][i][c + 2] * inv;
          }
        }
        __syncwarp();
        const int rows = min(8, static_cast<int>(w.group - r0) - 8 * x);  // one token
        for (int e = 2 * lane; e < rows * D; e += 64) {
          const int r = e / D, c = e % D;
          const float* v = own + r * L::kPad + c;
          *reinterpret_cast<uint32_t*>(out + done.s.first * ld_o +
                                       static_cast<int64_t>(hk * w.group + r0 + 8 * x + r) * (2 * D) +
                                       2 * c) = pack2<DT>(v[0], v[1]);
        }
        __syncwarp();
      }
      if (!go_on) break;
      clear();
    } else {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], d);
          if (g == 0) s_m(warp, 8 * x + 2 * t4 + c) = m[x][c];
        }
      __syncthreads();
      const uint32_t hk = done.hr / done.s.row_tiles;
      const uint32_t r0 = (done.hr - hk * done.s.row_tiles) * NR;
      const int rows = min(NR, static_cast<int>(done.s.count * w.group - r0));
      // (the rings are done with when the CTA's last row tile ends)
      float* part = CLUSTER ? reinterpret_cast<float*>(smem)
                            : att_slot<D, NR>(ws, 2 * blockIdx.x + (first_rows ? 0 : 1));
      if (!CLUSTER && !go_on && tile0 == 0 && !whole && threadIdx.x == 0) {
        // the last key tile's unit is this many on from the CTA's end
        const uint64_t e = u1 - 1 + (done.s.tiles - 1 - done.tile);
        uint32_t c1 = static_cast<uint32_t>(e * ctas / total);
        while (att_first_unit(total, c1 + 1, ctas) <= e) ++c1;
        *note = {c1 - blockIdx.x + 1, first_rows ? 0u : 1u, done.s.first, hk, r0, rows, {0, 0}};
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = 8 * x + 2 * t4 + c;
          float top = s_m(0, r);
#pragma unroll
          for (int i = 1; i < kAttWarps; ++i) top = fmaxf(top, s_m(i, r));
          const float f = exp2_approx(m[x][c] - (top == -INFINITY ? 0.f : top));
          if (g == 0) s_f(warp, r) = l[x][c] * f;  // this warp's sum on the common scale
          float* dst = merge + (warp * 8 + 2 * t4 + c) * L::kPad;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            dst[16 * i + g] = o[x][i][c] * f;
            dst[16 * i + g + 8] = o[x][i][c + 2] * f;
          }
        }
        __syncthreads();
        for (int e = 2 * threadIdx.x; e < 8 * D; e += 64 * kAttWarps) {
          const int r = 8 * x + e / D, c = e % D;
          if (r >= rows) break;
          float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
          for (int i = 0; i < kAttWarps; ++i) {
            sum += s_f(i, r);
            const float2 v = *reinterpret_cast<const float2*>(merge + (i * 8 + e / D) * L::kPad + c);
            v0 += v.x;
            v1 += v.y;
          }
          if (whole) {
            const uint32_t tok = MULTI ? w.by_group.div(r0 + r) : 0;
            const float inv = sum != 0.f ? 1.f / sum : 0.f;
            *reinterpret_cast<uint32_t*>(out + (done.s.first + tok) * ld_o +
                                         static_cast<int64_t>(hk * w.group + r0 + r - tok * w.group) * (2 * D) +
                                         2 * c) = pack2<DT>(v0 * inv, v1 * inv);
          } else {
            *reinterpret_cast<float2*>(part + 2 * NR + r * D + c) = make_float2(v0, v1);
            if (c == 0) {
              float top = s_m(0, r);
#pragma unroll
              for (int i = 1; i < kAttWarps; ++i) top = fmaxf(top, s_m(i, r));
              part[r] = top;
              part[NR + r] = sum;
            }
          }
        }
        __syncthreads();
      }
      if (!go_on) break;
      first_rows = false;
      tile0 = 0;
      clear();
    }
  }
  cp_async_wait<0>();
  if constexpr (CLUSTER) {
    if (cluster == 1) return;
    // every CTA of the cluster joins its share of the row tile's elements
    float* own = reinterpret_cast<float*>(smem);
    if (left0 <= 0) {  // more CTAs than key tiles
      for (int e = threadIdx.x; e < NR * (D + 2); e += 32 * kAttWarps) own[e] = e < NR ? -INFINITY : 0.f;
    }
    cluster_sync_all();
    const uint32_t hk = at.hr / at.s.row_tiles, r0 = (at.hr - hk * at.s.row_tiles) * NR;
    const int rows = min(NR, static_cast<int>(at.s.count * w.group - r0));
    const uint32_t base = smem_u32(own);
    // the parts' maxima and sums here first, then their outputs
    float* ml = own + NR * (D + 2);  // [cluster][2 NR]
    for (uint32_t e = threadIdx.x; e < cluster * 2 * NR; e += 32 * kAttWarps)
      ml[e] = ld_shared_cluster_f32(map_shared_rank(base + 4 * (e % (2 * NR)), e / (2 * NR)));
    __syncthreads();
#pragma unroll 4
    for (int e = 2 * (threadIdx.x + 32 * kAttWarps * rank); e < rows * D; e += 64 * kAttWarps * cluster) {
      const int r = e / D, c = e % D;
      float top = -INFINITY, sum = 0.f, v0 = 0.f, v1 = 0.f;
      for (uint32_t i = 0; i < cluster; ++i) top = fmaxf(top, ml[2 * NR * i + r]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
      for (uint32_t i = 0; i < cluster; ++i) {
        const float k = exp2_approx(ml[2 * NR * i + r] - ref);
        const uint32_t src = map_shared_rank(base + 4 * (2 * NR + e), i);
        sum += ml[2 * NR * i + NR + r] * k;
        v0 += ld_shared_cluster_f32(src) * k;
        v1 += ld_shared_cluster_f32(src + 4) * k;
      }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      *reinterpret_cast<uint32_t*>(out + at.s.first * ld_o + static_cast<int64_t>(hk * w.group + r0 + r) * (2 * D) +
                                   2 * c) = pack2<DT>(v0 * inv, v1 * inv);
    }
    cluster_sync_all();  // no CTA leaves while another reads its part
  }
}

// Joins the parts of the row tiles whose keys were split: blockIdx.x is the CTA
// that began one, blockIdx.y deals out its rows. The parts' factors first, then
// their outputs: a warp takes every eighth part, a lane D / 32 dimensions.
constexpr int kJoinWarps = 8, kJoinRows = 8;

template <int DT, int D, int NR>
__global__ void __launch_bounds__(32 * kJoinWarps)
    attention_join_kernel(char* out, const FastDiv by_group, int64_t ld_o, char* ws) {
  using T = typename DType<DT>::T;
  constexpr int E = D / 32, kThreads = 32 * kJoinWarps;
  __shared__ float s_f[kAttMaxCtas], s_red[kJoinWarps], s_v[kJoinWarps][D];
  pdl_launch_dependents();
  pdl_wait();
  const AttNote note = reinterpret_cast<const AttNote*>(ws)[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto slot = [&](uint32_t i) {
    return att_slot<D, NR>(ws, 2 * (blockIdx.x + i) + (i == 0 ? note.late : 0u));
  };
  if (note.parts == 0) return;
  for (int r = blockIdx.y; r < note.rows; r += kJoinRows) {
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < note.parts; i += kThreads) {
      const float m = slot(i)[r];
      s_f[i] = m;
      top = fmaxf(top, m);
    }
    top = block_reduce<true>(top, s_red);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (uint32_t i = threadIdx.x; i < note.parts; i += kThreads) {
      const float k = exp2_approx(s_f[i] - base);
      s_f[i] = k;
      sum += slot(i)[NR + r] * k;
    }
    sum = block_reduce<false>(sum, s_red);  // (its barriers publish s_f too)
    float v[E] = {};
#pragma unroll 4
    for (uint32_t i = warp; i < note.parts; i += kJoinWarps) {
      const float* p = slot(i) + 2 * NR + r * D + E * lane;
      const float k = s_f[i];
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] += x.x * k, v[1] += x.y * k, v[2] += x.z * k, v[3] += x.w * k;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] += x.x * k, v[1] += x.y * k;
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) s_v[warp][E * lane + k] = v[k];
    __syncthreads();
    if (threadIdx.x < D) {
      float o = 0.f;
#pragma unroll
      for (int k = 0; k < kJoinWarps; ++k) o += s_v[k][threadIdx.x];
      const uint32_t row = note.r0 + r, tok = by_group.div(row), group = by_group.d;
      T* dst = reinterpret_cast<T*>(out + (note.first + tok) * ld_o +
                                    static_cast<int64_t>(note.hk * group + row - tok * group) * (2 * D));
      dst[threadIdx.x] = DType<DT>::from_f32(sum != 0.f ? o / sum : 0.f);
    }
    __syncthreads();  // s_f and s_v are written again
  }
}

constexpr float kLog2e = 1.4426950408889634f;

inline AttWork att_work(const AttentionProblem& p, const PagedView& kv, uint32_t row_tile,
                        bool shared) {
  AttWork w;
  w.kv = kv;
  w.tokens = static_cast<uint32_t>(p.tokens);
  w.group = static_cast<uint32_t>(p.n_q / kv.n_kv);
  w.row_tile = row_tile;
  w.by_group = FastDiv(w.group);
  w.window = p.window;
  w.sinks = p.sinks;
  w.shared = shared;
  return w;
}

// Most units that a call can have, from what the host knows (the table's width).
inline uint64_t att_most_units(size_t batch, size_t tokens, size_t group, size_t n_kv, size_t keys,
                               size_t nr, bool multi) {
  const uint64_t tiles = std::max<uint64_t>(1, (keys + kAttKeys - 1) / kAttKeys) + kAttRowCost;
  const uint64_t row_tiles = multi ? std::min<uint64_t>(tokens * group, (tokens * group) / nr + batch)
                                   : batch * ((group + nr - 1) / nr);
  return tiles * row_tiles * n_kv;
}

// What the host knows of a call with one token per sequence: its row tiles, and
// the most keys that one can have by the table (or the window).
struct AttBounds {
  uint64_t row_tiles, keys;
};
inline AttBounds att_bounds(const AttentionProblem& p, const PagedView& kv, uint32_t nr) {
  const uint64_t group = p.n_q / kv.n_kv;
  AttBounds b = {static_cast<uint64_t>(kv.batch) * kv.n_kv * ((group + nr - 1) / nr),
                 static_cast<uint64_t>(kv.width) * kv.page.d};
  if (p.window > 0) b.keys = std::min<uint64_t>(b.keys, static_cast<uint64_t>(p.window) + p.sinks);
  return b;
}

// CTAs of a cluster per row tile, for calls that need no more than two waves of
// them and give none more than kAttClusterTiles key tiles; 0 for the others. One
// launch that joins in shared memory, or has nothing to join, against two: 1
// sequence of 1000 tokens, 32 heads, f16, 6.8 against 9.5 us (c = 8); 250
// sequences of 500 tokens, 16 / 1 heads, 17.5 against 33.6, of 1 to 500 tokens
// 12.4 against 18.6 (c = 1). Long or ragged batches need the dealt-out units:
// 32 sequences of 1 to 1000 tokens, 32 / 8 heads, 17.0 against 13.9.
// Several CTAs pay from four key tiles on (1 sequence of 128 tokens: 4.2 us with
// one, 4.9 with two; of 250: 5.7 and, with four, 5.1).
inline uint32_t att_cluster(const AttBounds& b, int sm_count) {
  const uint64_t tiles = (b.keys + kAttKeys - 1) / kAttKeys, wave = 2ull * sm_count;
  uint32_t c = kAttMaxCluster;
  while (c > 1 && (b.row_tiles * c > wave || c >= 2 * tiles || tiles < 4)) c /= 2;
  if (tiles > c * kAttClusterTiles || b.row_tiles > 2 * wave) return 0;
  return b.row_tiles <= wave || b.keys > kAttEachFew ? c : 0;
}

// Otherwise a warp per row tile where no row tile has many keys: no joins at
// all. us a call against the dealt-out units (bf16, D = 128, 32 / 8 heads): 256
// sequences of 16 / 128 / 250 tokens 7.3 / 25.9 / 44.4 against 19.2 / 35.4 /
// 52.9. Above kAttEachKeys the longest sequence's one warp is what the call
// waits for: 256 sequences of 1 to 1000 tokens 63.9 against 41.2. The same
// holds above kAttEachFew where the row tiles leave half the warps idle: 64
// sequences of 1 to 250 tokens 14.6 against 9.4 with a CTA for each, of 64
// tokens 5.8 against 7.2.
inline bool att_each(const AttBounds& b) {
  return b.keys <= kAttEachKeys && b.row_tiles < (1ull << 30);
}

template <int DT, int D, int NT>
cudaError_t launch_attention_cluster_t(const AttentionProblem& p, const PagedView& kv,
                                       uint32_t cluster) {
  static uint64_t done = 0;
  auto kern = attention_split_kernel<DT, D, NT, false, kAttCluster>;
  if (!(p.device < 64 && (done >> p.device & 1))) {
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                               cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = allow_smem(kern, AttLayout<D>::kSmem, p.device, &done);
  if (e != cudaSuccess) return e;
  AttWork w = att_work(p, kv, 8 * NT, false);
  const char* q = static_cast<const char*>(p.q);
  char *out = static_cast<char*>(p.out), *ws = nullptr;
  int64_t ld_q = static_cast<int64_t>(p.ld_q) * 2, ld_o = static_cast<int64_t>(p.ld_out) * 2;
  float sl = p.scale * kLog2e;
  void* a[] = {&q, &out, &w, &ld_q, &ld_o, &sl, &ws};
  const uint32_t row_tiles = kv.batch * kv.n_kv * ((w.group + 8 * NT - 1) / (8 * NT));
  return launch_pdl(kern, dim3(row_tiles * cluster), 32 * kAttWarps, AttLayout<D>::kSmem, p.stream, a,
                    cluster);
}

template <int DT, int D, int NT>
cudaError_t launch_attention_each_t(const AttentionProblem& p, const PagedView& kv) {
  static uint64_t done = 0;
  auto kern = attention_split_kernel<DT, D, NT, false, kAttEach>;
  const cudaError_t e = allow_smem(kern, AttLayout<D>::kSmem, p.device, &done);
  if (e != cudaSuccess) return e;
  AttWork w = att_work(p, kv, 8 * NT, false);
  const char* q = static_cast<const char*>(p.q);
  char *out = static_cast<char*>(p.out), *ws = nullptr;
  int64_t ld_q = static_cast<int64_t>(p.ld_q) * 2, ld_o = static_cast<int64_t>(p.ld_out) * 2;
  float sl = p.scale * kLog2e;
  void* a[] = {&q, &out, &w, &ld_q, &ld_o, &sl, &ws};
  const uint64_t items = static_cast<uint64_t>(kv.batch) * kv.n_kv * ((w.group + 8 * NT - 1) / (8 * NT));
  const uint32_t ctas = static_cast<uint32_t>(
      std::min<uint64_t>((items + kAttWarps - 1) / kAttWarps, 2 * p.sm_count));
  return launch_pdl(kern, dim3(ctas), 32 * kAttWarps, AttLayout<D>::kSmem, p.stream, a);
}

template <int DT, int D, int NT, bool MULTI>
cudaError_t launch_attention_split_t(const AttentionProblem& p, const PagedView& kv,
                                     bool shared) {
  static uint64_t done = 0;  // a lost update only repeats the call
  auto kern = attention_split_kernel<DT, D, NT, MULTI, kAttDealt>;
  cudaError_t e = allow_smem(kern, AttLayout<D>::kSmem, p.device, &done);
  if (e != cudaSuccess) return e;
  AttWork w = att_work(p, kv, 8 * NT, shared);
  const size_t keys = static_cast<size_t>(kv.width) * kv.page.d;
  const uint64_t most = att_most_units(kv.batch, p.tokens, w.group, kv.n_kv, keys, 8 * NT, MULTI);
  uint32_t ctas = static_cast<uint32_t>(
      std::min<uint64_t>(most, std::min(2 * p.sm_count, kAttMaxCtas)));
  const char* q = static_cast<const char*>(p.q);
  char* out = static_cast<char*>(p.out);
  int64_t ld_q = static_cast<int64_t>(p.ld_q) * 2, ld_o = static_cast<int64_t>(p.ld_out) * 2;
  float sl = p.scale * kLog2e;
  char* ws = static_cast<char*>(p.workspace);
  void* a[] = {&q, &out, &w, &ld_q, &ld_o, &sl, &ws};
  e = launch_pdl(kern, dim3(ctas), 32 * kAttWarps, AttLayout<D>::kSmem, p.stream, a);
  // no row tile can be split: its keys fit one unit
  if (e != cudaSuccess || keys <= kAttKeys || ctas == 1) return e;
  FastDiv by_group = w.by_group;
  void* b[] = {&out, &by_group, &ld_o, &ws};
  return launch_pdl(attention_join_kernel<DT, D, 8 * NT>, dim3(ctas - 1, kJoinRows),
                    32 * kJoinWarps, 0, p.stream, b);
}

inline size_t att_row_tile(size_t group, bool multi) { return multi || group > 8 ? 16 : 8; }

inline size_t attention_split_workspace(size_t batch, size_t tokens, size_t group, size_t n_kv,
                                        size_t keys, size_t d, bool multi) {
  const size_t nr = att_row_tile(group, multi);
  const uint64_t most = att_most_units(batch, tokens, group, n_kv, keys, nr, multi);
  return kAttNotes + std::min<uint64_t>(most, kAttMaxCtas) * 2 * nr * (d + 2) * sizeof(float);
}

cudaError_t launch_attention_split(const AttentionProblem& p, const PagedView& kv,
                                   bool shared) {
  const bool multi = kv.q_start != nullptr;
  const bool two = att_row_tile(p.n_q / kv.n_kv, multi) == 16;
  const AttBounds bounds = att_bounds(p, kv, two ? 16 : 8);
  const uint32_t cluster = multi ? 0 : att_cluster(bounds, p.sm_count);
  const bool each = !multi && cluster == 0 && att_each(bounds);
#define CAWQ_ATT(DT, D)                                                              \
  (each ? two ? launch_attention_each_t<DT, D, 2>(p, kv)                             \
              : launch_attention_each_t<DT, D, 1>(p, kv)                             \
   : cluster ? two ? launch_attention_cluster_t<DT, D, 2>(p, kv, cluster)            \
                   : launch_attention_cluster_t<DT, D, 1>(p, kv, cluster)            \
   : multi ? launch_attention_split_t<DT, D, 2, true>(p, kv, shared)                 \
         : two ? launch_attention_split_t<DT, D, 2, false>(p, kv, shared)          \
               : launch_attention_split_t<DT, D, 1, false>(p, kv, shared))
  if (p.dtype == kF16) return p.d == 64 ? CAWQ_ATT(kF16, 64) : CAWQ_ATT(kF16, 128);
  return p.d == 64 ? CAWQ_ATT(kBF16, 64) : CAWQ_ATT(kBF16, 128);
#undef CAWQ_ATT
}

}  // namespace cawq
