// Decode attention over the paged KV cache for sequences that share the beginning of their contexts.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// prefix_attention_kernel, prefix_join_kernel
//
// Softmax over a context is the join of softmaxes over its pieces: with maxima m_k, sums l_k and unnormalised results O_k of the pieces,
// O = sum w_k O_k / sum w_k l_k, w_k = exp(m_k - max m).  So the common beginning of a group's contexts is walked once for all of its sequences, whose
// query heads fill the 128 rows of the tensor core, and the rest of each context for its own.
//
// The common keys are those that every sequence of the group has, in whole tiles of 64, so that no row of theirs is masked.  The two kinds of keys are walked by different warps of
// a CTA, one CTA per SM, because they are bound by different things and go on beside each other.  Others are bound by HBM: 256 contexts of 3000 tokens, 64 / 8 heads of 128, 508 us or
// 6.2 TB/s, of 375 tokens (an item every six tiles) 4.9.  Common ones take 0.9 to 1 us a tile of 128 rows x 64 keys, 131 us for 256 sequences behind 8192 tokens, 64 / 8 heads: none of tensor core
// (28 %), exponentials (30 %) and issue slots (27 %) is full, and the copies of a tile take 2500 clocks to arrive.  One thread per row in place of two took 143 us, and with blocks of 16 tokens 41 us in place
// of 31 for a ragged batch; scores and results by a warp each 148; three stages for the common keys and two for the others 129 and, for the others, 164 in place of 145.
//
// Of each kind, the tiles of all items are dealt in contiguous equal ranges to the CTAs, from lengths that are read on the device, so that a captured call stays balanced for any
// batch.  A piece that begins an item is left in a row of its own, one for common and one for other keys, a piece that goes on with one that an earlier range
// began in the range's slot; prefix_join_kernel joins them.  Sequences without common keys whose context is one piece are stored at once.
// ---------------------------------------------------------------------------
constexpr int PX_ROWS = 128, PX_KEYS = 64, PX_COLUMNS = 512;
constexpr int PX_WARPS = 10, PO_WARPS = 4, PX_THREADS = (PX_WARPS + PO_WARPS + 1) * 32;  // of common keys, of others and their TMA warp
constexpr int PX_MAX_SEQS = 1024, PX_MAX_GROUPS = 512;
constexpr int PX_ITEM_UNITS = 2;  // what an item costs beside its tiles, in tiles
constexpr int PX_WHOLE_TILES = 8;
constexpr float PX_GROWTH = 8.f;
constexpr uint64_t PX_LIMIT_NS = 1000000000ull;

template <int HD>
struct Prefix {
  static constexpr int HALVES = HD / 64;
  static constexpr int STAGES = 4 / HALVES;  // tiles of K, and as many of V
  static constexpr uint32_t HALF = PX_KEYS * 128;  // 64 keys of 64 dimensions: one swizzled box
  static constexpr uint32_t TILE = HALVES * HALF;
  static constexpr uint32_t Q_HALF = PX_ROWS * 128;
  static constexpr uint32_t Q = HALVES * Q_HALF;
  static constexpr int SLOT = PX_ROWS * (HD + 2);  // floats of a range's piece: O as [HD / 4][row][4], then the maxima and the sums
  // the other keys: tiles of K and V side by side, each stage with room for Q where a segment begins, and the warps' results where they meet, a pad after each row
  static constexpr int OWN_STAGES = 6 / HALVES, OWN_ROWS = 16, OWN_SLOT = OWN_ROWS * (HD + 2);
  static constexpr uint32_t OWN_RING = Q + 2 * STAGES * TILE, OWN_Q = OWN_RING + OWN_STAGES * 2 * TILE;
  __host__ __device__ static constexpr uint32_t own_q(int h) { return h * 1024 * HALVES; }  // 8 h rows
  __host__ __device__ static constexpr int meet_dims(int h) { return h == 1 ? 64 : 32; }    // dimensions that meet at a time
  __host__ __device__ static constexpr uint32_t meet(int h) { return OWN_Q + OWN_STAGES * own_q(h); }
  __host__ __device__ static constexpr uint32_t plan(int h) { return meet(h) + PO_WARPS * 8 * h * (meet_dims(h) + 4) * 4; }
  static constexpr size_t smem(int h, int n_seqs, int n_groups) { return 1024 + plan(h) + (2 * n_groups + n_seqs + 2) * sizeof(int) + n_seqs * sizeof(uint16_t); }
};
constexpr size_t PX_STATIC = 2944, PX_SMEM = 227 * 1024;
static_assert(Prefix<128>::smem(1, PX_MAX_SEQS, PX_MAX_GROUPS) + PX_STATIC <= PX_SMEM && Prefix<128>::smem(2, PX_MAX_SEQS, PX_MAX_GROUPS) + PX_STATIC <= PX_SMEM &&
                  Prefix<64>::smem(1, PX_MAX_SEQS, PX_MAX_GROUPS) + PX_STATIC <= PX_SMEM && Prefix<64>::smem(2, PX_MAX_SEQS, PX_MAX_GROUPS) + PX_STATIC <= PX_SMEM,
              "a CTA's shared memory");

struct PrefixArgs {
  const int32_t* tables;
  int64_t bt_stride;
  int bt_width, block_size, num_blocks, box;  // box: rows of a tensor map's box, which lie inside one block
  const int32_t *cu, *prefix, *lens;
  int n_groups, n_seqs, nq, nkv, group, npt, row_blocks;  // group: query heads per KV head; npt: sequences of 128 rows; row_blocks: 16 heads of a group each
  uint32_t negate;                // the instruction descriptor's bit that negates Q, where the scale is negative
  float scale_log2, signed_log2;  // softmax scale * log2(e): its size, itself
  uint16_t* out;
  // pieces that begin an item: [2][HD / 4][rows][4], maxima (as exponents of two) [2][rows], sums [2][rows] for common and other keys; rows: (KV head, sequence,
  // head of its group)
  float *rows_o, *rows_m, *rows_l;
  float *slots, *own_slots;  // [ranges]
  int ranges;
  int* plan;   // for the join
  bool whole;  // every (sequence, KV head, 16 heads) is one CTA's, from its first key on: there are no pieces
  B2Status* status;
};

// What the batch's lengths come to, in shared memory or in the workspace.
struct Plan {
  int *common_units;  // [n_groups + 1] units of the common keys of the groups before each
  int *common;        // [n_groups] tiles of common keys, times 1024, and the sequence whose table has them
  int *own_units;     // [n_seqs + 1] units of the other keys
  uint16_t* group_of; // [n_seqs]; 0xffff: none
  __device__ __forceinline__ int common_tiles(int g) const { return common[g] >> 10; }
  __device__ __forceinline__ int leader(int g) const { return common[g] & 1023; }
};
__device__ __forceinline__ Plan plan_of(int* at, int n_groups, int n_seqs) {
  return {at, at + n_groups + 1, at + 2 * n_groups + 1, reinterpret_cast<uint16_t*>(at + 2 * n_groups + n_seqs + 2)};
}
__device__ __forceinline__ int length(const PrefixArgs& a, int s) { return max(0, min(__ldg(a.lens + s), a.bt_width * a.block_size)); }
__device__ __forceinline__ int bound(const PrefixArgs& a, int g) { return max(0, min(__ldg(a.cu + g), a.n_seqs)); }
__device__ __forceinline__ int tiles_of(int keys) { return (keys + PX_KEYS - 1) / PX_KEYS; }
__device__ __forceinline__ int last_at(const int* first, int n, int unit) {  // the last that begins at or before the unit
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= unit) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// All threads of a block fill the plan; scratch: [n_groups] ints of shared memory that the async proxy writes later.
__device__ __forceinline__ void make_plan(const PrefixArgs& a, const Plan& plan, int* first_live) {
  const int n_seqs = a.n_seqs, n_groups = a.n_groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool falls = false;  // bounds that fall: groups would overlap, and their rows' pieces too
  for (int g = threadIdx.x; g < n_groups; g += PX_THREADS) {
    first_live[g] = PX_MAX_SEQS;
    plan.common[g] = max(0, __ldg(a.prefix + g));
    const int from = bound(a, g), to = bound(a, g + 1);
    falls = falls || to < from;
    plan.common_units[g + 1] = to;  // (for the search below)
    if (g == 0) plan.common_units[0] = from;
  }
  falls = __syncthreads_or(falls) != 0;
  for (int s = threadIdx.x; s < n_seqs; s += PX_THREADS) {
    const int len = length(a, s);
    int g = last_at(plan.common_units, n_groups, s);
    if (n_groups == 0 || falls || s < plan.common_units[g] || s >= plan.common_units[g + 1]) g = 0xffff;
    plan.group_of[s] = static_cast<uint16_t>(g);
    if (g != 0xffff && len > 0) {  // (a sequence without tokens shortens nothing, and its table may be anything)
      atomicMin(plan.common + g, len);
      atomicMin(first_live + g, s);
    }
  }
  __syncthreads();
  for (int g = threadIdx.x; g < n_groups; g += PX_THREADS) {
    // a group of one has nothing in common with another one
    if (a.whole || plan.common_units[g + 1] - plan.common_units[g] < 2 || first_live[g] == PX_MAX_SEQS) plan.common[g] = 0;
    else plan.common[g] = (plan.common[g] / PX_KEYS) << 10 | first_live[g];
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  auto add_up = [&](int* sums, int n, auto units) {  // by one warp
    const int per = (n + 31) / 32, i0 = lane * per;
    int mine = 0;
    for (int i = i0; i < min(n, i0 + per); ++i) mine += units(i);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    int at = incl - mine;
    __syncwarp();
    for (int i = i0; i < min(n, i0 + per); ++i) {
      const int all = units(i);
      sums[i + 1] = at += all;
    }
    if (lane == 0) sums[0] = 0;
  };
  if (warp == 0) {
    add_up(plan.common_units, n_groups, [&](int g) {
      const int n = bound(a, g + 1) - bound(a, g);
      return plan.common_tiles(g) > 0 ? a.nkv * ((n + a.npt - 1) / a.npt) * (plan.common_tiles(g) + PX_ITEM_UNITS) : 0;
    });
  } else if (warp == 1) {
    add_up(plan.own_units, n_seqs, [&](int s) {
      const int g = plan.group_of[s], keys = g == 0xffff ? 0 : length(a, s) - plan.common_tiles(g) * PX_KEYS;
      return keys > 0 ? a.nkv * a.row_blocks * (tiles_of(keys) + PX_ITEM_UNITS) : 0;
    });
  }
}

// Ranges of `total` units: x of X
struct Deal {
  int ctas, base, rem;
  __device__ __forceinline__ Deal(int total, int X) {
    const int per = (total + X - 1) / X;
    ctas = min(X, per <= PX_ITEM_UNITS + 6 ? (total + max(1, per) - 1) / max(1, per) : X);
    base = ctas > 0 ? total / ctas : 0;
    rem = ctas > 0 ? total % ctas : 0;
  }
  __device__ __forceinline__ int begin_of(int x) const { return x < ctas ? x * base + min(x, rem) : 0; }
  __device__ __forceinline__ int end_of(int x) const { return x < ctas ? begin_of(x) + base + (x < rem ? 1 : 0) : 0; }
  __device__ __forceinline__ int cta_of(int t) const {
    const int big = rem * (base + 1);
    return t < big ? t / (base + 1) : rem + (t - big) / base;
  }
};

// A segment: tiles t0 .. t1 of an item with `tiles` of them, which begin at key `start` of a context of `len` keys in the blocks of sequence `table`.  Its rows:
// `rows` from row `row` of sequence seq's group of heads on.
struct Segment {
  int seq, head, row, rows, table, start, len, tiles, t0, t1;
};
// A range [pos, end) of units as segments that lie inside one item.  An item has a unit for each of its tiles and, before those, PX_ITEM_UNITS for its beginning
// and its end.  A segment may hold no tiles (t0 >= t1).
template <bool OWN>
struct PrefixWalk {
  const Plan plan;
  int pos, end, at, known;  // at: group or sequence; known: the one that the segment is of
  __device__ __forceinline__ PrefixWalk(const PrefixArgs& a, const Plan& p, int begin, int stop) : plan(p), pos(begin), end(stop), known(-1) {
    at = last_at(OWN ? plan.own_units : plan.common_units, OWN ? a.n_seqs : a.n_groups, pos);
  }
  __device__ __forceinline__ bool next(const PrefixArgs& a, Segment& x) {
    if (pos >= end) return false;
    const int* first = OWN ? plan.own_units : plan.common_units;
    while (first[at + 1] <= pos) ++at;
    if (at != known) {  // (the items of a sequence, or of a group, lie one after the other)
      known = at;
      if (OWN) {
        x.len = length(a, at);
        x.start = plan.common_tiles(plan.group_of[at]) * PX_KEYS;
        x.tiles = tiles_of(x.len - x.start);
        x.table = x.seq = at;
      } else {
        x.start = 0;
        x.tiles = plan.common_tiles(at);
        x.len = x.tiles * PX_KEYS;
        x.table = plan.leader(at);
      }
    }
    const int units = x.tiles + PX_ITEM_UNITS, in = pos - first[at], item = in / units, u0 = in - item * units;
    if (OWN) {
      x.head = item / a.row_blocks;
      x.row = (item - x.head * a.row_blocks) * 16;
      x.rows = min(16, a.group - x.row);
    } else {
      const int begin = bound(a, at), n = bound(a, at + 1) - begin, high = (n + a.npt - 1) / a.npt;
      x.head = item / high;
      const int y = item - x.head * high;
      x.seq = begin + y * a.npt;
      x.row = 0;
      x.rows = min(a.npt, n - y * a.npt) * a.group;  // (of several sequences)
    }
    const int u1 = min(units, u0 + end - pos);
    pos += u1 - u0;
    x.t0 = max(0, u0 - PX_ITEM_UNITS);
    x.t1 = u1 - PX_ITEM_UNITS;
    // (Coordinates of TMA loads.  In registers of each thread, all of them with the same value, one of two loads of Q took another for its first coordinate: zeros.)
    x.seq = b2::uniform(x.seq);
    x.head = b2::uniform(x.head);
    x.row = b2::uniform(x.row);
    return true;
  }
};

// Rows of the cache of a segment's boxes, 32 at a time, one per lane, and those of the next 32 before they are needed: an entry of the table takes half a
// microsecond to arrive.
struct BoxRows {
  const PrefixArgs& a;
  const int32_t* table;
  int first, last, rows, next, group;
  __device__ __forceinline__ BoxRows(const PrefixArgs& args, const Segment& s) : a(args), table(args.tables + static_cast<int64_t>(s.table) * args.bt_stride), group(0) {
    first = s.start / a.box + s.t0 * (PX_KEYS / a.box);
    last = (s.len + a.box - 1) / a.box;
    rows = of(0);
    next = of(1);
  }
  __device__ __forceinline__ int of(int g) const {
    const int box = first + g * 32 + static_cast<int>(threadIdx.x & 31), p = box * a.box, blk = p / a.block_size;
    if (box >= last) return 0;
    return min(max(0, __ldg(table + blk)), a.num_blocks - 1) * a.block_size + p - blk * a.block_size;  // inside the cache whatever the table holds
  }
  // boxes i .. i + 3 of the segment's, in order; those of a tile, so that they do not go past a multiple of 32 (what is behind the tile's means nothing)
  __device__ __forceinline__ void four(int i, int (&r)[4]) {
    if (i >> 5 != group) {
      rows = next;
      group = i >> 5;
      next = of(group + 1);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = __shfl_sync(0xffffffffu, rows, (i + k) & 31);
  }
};

// ---- the common keys: 128 rows of the tensor core -----------------------------------------------------------------------------------------
//   warps 0..7   two threads per row, one for the even and one for the odd tiles, each with its own running maximum, sum and O: P = exp2(...) rounded to bf16 over the scores
//                in tensor memory (the product's operand has 16 bits), and O rescaled where the maximum has grown.  They meet at the segment's end.
//   warp 8       TMA: Q of the segment, then K and V tiles
//   warp 9       tcgen05.mma: S = Q K^T (128 x 64, four buffers), O += P V with P read from tensor memory
template <int HD>
__device__ __forceinline__ void common_keys(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const PrefixArgs& a, const Plan& plan, uint32_t s_q, uint32_t bars, uint32_t tmem,
                                            float (*s_m)[PX_ROWS], float (*s_l)[PX_ROWS], int warp, volatile int* abort_flag) {
  using T = Prefix<HD>;
  constexpr int HALVES = T::HALVES, STAGES = T::STAGES;
  const uint32_t s_k = s_q + T::Q, s_v = s_k + STAGES * T::TILE;
  const uint32_t q_full = bars, q_empty = q_full + 8, k_full = q_empty + 8, k_empty = k_full + STAGES * 8, v_full = k_empty + STAGES * 8, v_empty = v_full + STAGES * 8,
                 s_full = v_empty + STAGES * 8, p_full = s_full + 4 * 8, o_done = p_full + 4 * 8, met = o_done + 4 * 8;
  const int lane = threadIdx.x & 31, x = blockIdx.x;
  const Deal deal(plan.common_units[a.n_groups], gridDim.x);
  const int begin = deal.begin_of(x), end = deal.end_of(x);
  PrefixWalk<false> walk(a, plan, begin, end);
  Segment seg;
  auto all_wait = [&](uint32_t bar, uint32_t phase, int code) {
    return __all_sync(0xffffffffu, b2::mbar_wait(bar, phase, abort_flag, PX_LIMIT_NS, code)) != 0;
  };
  int c = 0, segs = 0;  // tiles and segments so far

  if (begin >= end) {
  } else if (warp == 8) {
    // ---------------- TMA (the whole warp walks and one thread issues, here and in the next warp) ----------------
    bool ok = true;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      ok = all_wait(q_empty, (segs & 1) ^ 1, B2_WAIT_SMEM_EMPTY);
      if (!ok) break;
      if (b2::elect_one()) {
        b2::mbar_arrive_expect_tx(q_full, HALVES * 128 * a.group * a.npt);
        for (int i = 0; i < HALVES; ++i) b2::tma_load_3d(s_q + i * T::Q_HALF, &tmQ, q_full, i * 64, seg.head * a.group, seg.seq, b2::kEvictNormal);
      }
      __syncwarp();
      // (K runs ahead of V, which keeps its own rows)
      const int per_tile = PX_KEYS / a.box;
      BoxRows k_rows(a, seg), v_rows = k_rows;
      auto load = [&](int j, int no, const CUtensorMap* map, uint32_t full, uint32_t empty, uint32_t dst, BoxRows& rows) {
        const int st = no % STAGES;
        if (!all_wait(empty + st * 8, ((no / STAGES) & 1) ^ 1, B2_WAIT_SMEM_EMPTY)) return false;
        const uint32_t bar = full + st * 8;
        int r[4];
        rows.four(j * per_tile, r);
        if (b2::elect_one()) {  // (one after the other by one thread: an election for each box took 0.1 us more)
          b2::mbar_arrive_expect_tx(bar, T::TILE);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < per_tile)
              for (int h = 0; h < HALVES; ++h) b2::tma_load_2d(dst + st * T::TILE + h * T::HALF + i * a.box * 128, map, bar, seg.head * HD + h * 64, r[i], b2::kEvictNormal);
        }
        __syncwarp();
        return true;
      };
      auto load_k = [&](int j) { return load(j, c + j, &tmK, k_full, k_empty, s_k, k_rows); };
      auto load_v = [&](int j) { return load(j, c + j, &tmV, v_full, v_empty, s_v, v_rows); };
      // in the order of use: K of three tiles, then V of a tile and K of the third after it
      const int n = seg.t1 - seg.t0;
      for (int j = 0; ok && j < min(n, 3); ++j) ok = load_k(j);
      for (int j = 0; ok && j < n; ++j) {
        ok = load_v(j);
        if (j + 3 < n) ok = ok && load_k(j + 3);
      }
      c += n;
      ++segs;
    }
  } else if (warp == 9) {
    // ---------------- tensor core ----------------
    const uint32_t idesc_s = b2::umma_idesc_bf16(PX_KEYS) | a.negate;
    constexpr uint32_t idesc_o = b2::umma_idesc_bf16(HD) | (1u << 16);  // second operand MN-major
    const uint64_t desc_q = b2::umma_smem_desc(s_q), desc_k = b2::umma_smem_desc(s_k), desc_v = b2::umma_smem_desc_mn(s_v, T::HALF);  // (addresses in 16 bytes)
    auto wait = [&](uint32_t bar, uint32_t phase, int code) {
      const bool ok = all_wait(bar, phase, code);
      b2::tc_fence_after();
      return ok;
    };
    // scores of tile i, into the columns that P of tile i - 4 was read from, once it has been
    auto scores = [&](int i, bool last) {
      const int st = i % STAGES, buf = i & 3;
      bool ok = i < 4 || wait(o_done + buf * 8, ((i >> 2) & 1) ^ 1, B2_WAIT_TMEM_FULL);
      ok = ok && wait(k_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL);
      if (ok && b2::elect_one()) {
        const uint64_t dk = desc_k + st * (T::TILE >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          b2::umma_bf16(tmem + buf * PX_KEYS, desc_q + (k >> 2) * (T::Q_HALF >> 4) + 2 * (k & 3), dk + (k >> 2) * (T::HALF >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
        b2::umma_commit(s_full + buf * 8);
        b2::umma_commit(k_empty + st * 8);
        if (last) b2::umma_commit(q_empty);
      }
      __syncwarp();
      return ok;
    };
    bool ok = true;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      const int n = seg.t1 - seg.t0;
      ok = wait(q_full, segs & 1, B2_WAIT_SMEM_FULL);
      for (int j = 0; ok && j < min(n, 3); ++j) ok = scores(c + j, j + 1 == n);
      for (int j = 0; ok && j < n; ++j) {
        const int i = c + j, st = i % STAGES, buf = i & 3;
        ok = wait(v_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL) && wait(p_full + buf * 8, (i >> 2) & 1, B2_WAIT_TMEM_EMPTY);
        if (!ok) break;
        if (b2::elect_one()) {
          const uint64_t dv = desc_v + st * (T::TILE >> 4);
#pragma unroll
          for (int k = 0; k < PX_KEYS / 16; ++k)  // 16 tokens: 8 columns of P, 2048 bytes of V
            b2::umma_bf16_ts(tmem + 4 * PX_KEYS + (i & 1) * HD, tmem + buf * PX_KEYS + k * 8, dv + k * (2048 >> 4), idesc_o, (j > 1 || k > 0) ? 1u : 0u);
          b2::umma_commit(o_done + buf * 8);
          b2::umma_commit(v_empty + st * 8);
        }
        __syncwarp();
        if (j + 3 < n) ok = scores(i + 3, j + 4 == n);
      }
      c += n;
      ++segs;
    }
  } else {
    // ---------------- two threads per row ----------------
    const int row = threadIdx.x & (PX_ROWS - 1), odd = warp >> 2;  // odd: which tiles
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, t_o = tmem + 4 * PX_KEYS + odd * HD + lanes;
    int meetings = 0;
    auto all_here = [&]() {  // the eight warps, like a barrier, but bounded
      b2::tc_fence_before();
      __syncwarp();
      if (lane == 0) b2::mbar_arrive(met);
      const bool here = all_wait(met, meetings & 1, B2_WAIT_TMEM_FULL);
      ++meetings;
      b2::tc_fence_after();
      return here;
    };
    const uint64_t scale2 = b2::pair_of(a.scale_log2, a.scale_log2);
    const int64_t all_rows = static_cast<int64_t>(a.n_seqs) * a.nq;
    bool ok = true;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      const int n = seg.t1 - seg.t0;
      float m = -INFINITY;  // the row's maximum, in units of scores
      uint64_t l[2] = {};   // its sum, in two pairs
      const bool idle = (warp & 3) * 32 >= seg.rows;  // none of the warp's rows exists
      for (int j = (c ^ odd) & 1; j < n; j += 2) {
        const int i = c + j, buf = i & 3;
        ok = all_wait(s_full + buf * 8, (i >> 2) & 1, B2_WAIT_TMEM_FULL);
        if (!ok) break;
        b2::tc_fence_after();
        if (!idle) {
          const uint32_t t_s = tmem + buf * PX_KEYS + lanes;
          uint32_t r[2][32];
          b2::tmem_ld_32x32(t_s, r[0]);
          b2::tmem_ld_32x32(t_s + 32, r[1]);
          b2::tc_wait_ld(r);
          float mx[4] = {m, m, m, m};
#pragma unroll
          for (int e = 0; e < 64; e += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], __uint_as_float(r[e >> 5][(e & 31) + k]));
          // The reference m moves when the row is PX_GROWTH past it (or has seen its first key): O then has to be rescaled, which takes as long as
          // half a tile.  Until then probabilities are up to 2^PX_GROWTH, rounded relative to themselves.  (Each row for itself: its result does not
          // depend on the rows beside it.)
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool grown = (top - m) * a.scale_log2 > PX_GROWTH;
          const float f = grown ? b2::ex2((m - top) * a.scale_log2) : 1.f;
          if (grown) m = top;
          const float ref = m == -INFINITY ? 0.f : m * a.scale_log2;
          const uint64_t ref2 = b2::pair_of(-ref, -ref);
          const bool any_grown = __any_sync(0xffffffffu, grown);
          if (any_grown) {
            l[0] = b2::mul_pair(l[0], b2::pair_of(f, f));
            l[1] = b2::mul_pair(l[1], b2::pair_of(f, f));
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float u, w;
              b2::fma_pair(u, w, b2::pair_of(__uint_as_float(r[h][e]), __uint_as_float(r[h][e + 1])), scale2, ref2);
              u = b2::ex2(u);
              w = b2::ex2(w);
              l[(e >> 1) & 1] = b2::add_pair(l[(e >> 1) & 1], b2::pair_of(u, w));
              p[e >> 1] = b2::pack_bf16(u, w);
            }
            b2::tmem_st_32x16(t_s + h * 16, p);  // (this row has read its columns)
          }
          if (j > 1 && any_grown) {
            ok = all_wait(o_done + ((i - 2) & 3) * 8, ((i - 2) >> 2) & 1, B2_WAIT_TMEM_FULL);
            if (!ok) break;
            b2::tc_fence_after();
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              b2::tmem_ld_32x32(t_o + h * 64, r[0]);
              b2::tmem_ld_32x32(t_o + h * 64 + 32, r[1]);
              b2::tc_wait_ld(r);
#pragma unroll
              for (int e = 0; e < 64; ++e) r[e >> 5][e & 31] = __float_as_uint(__uint_as_float(r[e >> 5][e & 31]) * f);
#pragma unroll
              for (int k = 0; k < 4; ++k) b2::tmem_st_32x16(t_o + h * 64 + k * 16, &r[k >> 1][(k & 1) * 16]);
            }
          }
          b2::tc_wait_st();
        }
        b2::tc_fence_before();
        __syncwarp();
        if (lane == 0) b2::mbar_arrive(p_full + buf * 8);
      }
      if (!ok) break;
      // ---- both threads' results together ----
      const int first = (c ^ odd) & 1, last = c + n - 1 - ((n - 1 - first) & 1);  // of this thread's tiles, if it has any
      if (first < n) ok = all_wait(o_done + (last & 3) * 8, (last >> 2) & 1, B2_WAIT_TMEM_FULL);
      if (!ok) break;
      if (!idle) {
        float sums[2];
        b2::halves_of(b2::add_pair(l[0], l[1]), sums[0], sums[1]);
        s_m[odd][row] = m;
        s_l[odd][row] = sums[0] + sums[1];
      }
      ok = all_here();
      if (!ok) break;
      if (!idle) {
        const bool exists = row < seg.rows, begins = seg.t0 == 0;
        const float m0 = s_m[0][row], m1 = s_m[1][row], top = fmaxf(m0, m1);
        // (one tile: the other O holds anything)
        const float f0 = m0 == top ? 1.f : b2::ex2((m0 - top) * a.scale_log2), f1 = m1 == top ? 1.f : b2::ex2((m1 - top) * a.scale_log2);
        const bool has0 = n > 1 || (c & 1) == 0, has1 = n > 1 || (c & 1) == 1;
        const int64_t at = (static_cast<int64_t>(seg.head) * a.n_seqs + seg.seq) * a.group + row;  // (sequences of 128 rows lie one after the other)
        float* const slot = a.slots + static_cast<int64_t>(x) * T::SLOT;
        float* const o = begins ? a.rows_o + at * 4 : slot + row * 4;
        const int64_t step = begins ? all_rows * 4 : PX_ROWS * 4;
#pragma unroll
        for (int d0 = 0; d0 < HD / 2; d0 += 32) {  // each of the two brings half of the dimensions
          const int d = odd * (HD / 2) + d0;
          uint32_t r[2][32];
          b2::tmem_ld_32x32(tmem + 4 * PX_KEYS + lanes + d, r[0]);
          b2::tmem_ld_32x32(tmem + 4 * PX_KEYS + HD + lanes + d, r[1]);
          b2::tc_wait_ld(r);
          if (exists) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] = (has0 ? __uint_as_float(r[0][e + k]) * f0 : 0.f) + (has1 ? __uint_as_float(r[1][e + k]) * f1 : 0.f);
              *reinterpret_cast<float4*>(o + (d + e) / 4 * step) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
          __syncwarp();
        }
        if (exists && odd == 0) {
          (begins ? a.rows_m + at : slot + HD * PX_ROWS + row)[0] = top * a.scale_log2;
          (begins ? a.rows_l + at : slot + (HD + 1) * PX_ROWS + row)[0] = (has0 ? s_l[0][row] * f0 : 0.f) + (has1 ? s_l[1][row] * f1 : 0.f);
        }
      }
      ok = all_here();  // (the next segment's products write over O)
      c += n;
      ++segs;
    }
  }

}

// ---- the other keys: up to 16 heads of one sequence -----------------------------------------------------------------------------------------
// Every K and V row is used by the heads of one group only, which would fill a fraction of the tensor core's 128 rows: mma.sync with the keys (of the scores, S^T = K Q^T) and
// the dimensions (of the result, O^T = V^T P^T) on its 16 rows and 8 heads on its columns does as much work as there is.  Bound: HBM; a warp's chain of products and exponentials
// is 0.6 of a tile's time on it.
//   warps 0..3   16 keys of each tile of 64, each warp with its own maxima, sums and results, which meet at the segment's end
//   warp 4       TMA: K and V tiles, Q with the first
__device__ __forceinline__ void mma_16x8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a warp's 8 x 8 matrix of 16-bit numbers, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// H: times 8 heads; warp: of these
template <int HD, int H>
__device__ __forceinline__ void own_keys(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const PrefixArgs& a, const Plan& plan, unsigned char* smem, uint32_t bars, float (*s_m)[16],
                                         float (*s_l)[16], int warp, volatile int* abort_flag) {
  using T = Prefix<HD>;
  constexpr int HALVES = T::HALVES, STAGES = T::OWN_STAGES, STEPS = HD / 16, DIMS = T::meet_dims(H), PAD = DIMS + 4;
  const uint32_t base = b2::smem_u32(smem), ring = base + T::OWN_RING, s_q = base + T::OWN_Q;
  float* const meet = reinterpret_cast<float*>(smem + T::meet(H));  // [PO_WARPS][8 H][PAD]
  const uint32_t full = bars, empty = full + STAGES * 8, met = empty + STAGES * 8;
  const int lane = threadIdx.x & 31, tid = warp * 32 + lane, x = blockIdx.x;
  int begin, end;
  if (a.whole) {  // CTA x is item x
    const int items = a.nkv * a.row_blocks, s = x / items, i = x - s * items, units = (plan.own_units[s + 1] - plan.own_units[s]) / items;
    begin = plan.own_units[s] + i * units;
    end = begin + units;
    if (units == 0) {  // nothing to see
      const int head = i / a.row_blocks, row = (i - head * a.row_blocks) * 16, rows = min(16, a.group - row);
      uint4* out = reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(s) * a.nq + head * a.group + row) * HD);
      for (int e = tid; e < rows * HD / 8; e += (PO_WARPS + 1) * 32) out[e] = make_uint4(0, 0, 0, 0);
    }
  } else {
    const Deal deal(plan.own_units[a.n_seqs], gridDim.x);
    begin = deal.begin_of(x);
    end = deal.end_of(x);
    if (x == 0) {  // for the join
      const int words = 2 * a.n_groups + a.n_seqs + 2 + (a.n_seqs + 1) / 2;
      for (int i = tid; i < words; i += (PO_WARPS + 1) * 32) a.plan[i] = plan.common_units[i];
    }
  }
  PrefixWalk<true> walk(a, plan, begin, end);
  Segment seg;
  auto all_wait = [&](uint32_t bar, uint32_t phase, int code) {
    return __all_sync(0xffffffffu, b2::mbar_wait(bar, phase, abort_flag, PX_LIMIT_NS, code)) != 0;
  };
  int c = 0;  // tiles so far
  bool ok = true;

  if (begin >= end) {
  } else if (warp == PO_WARPS) {
    const int per_tile = PX_KEYS / a.box;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      BoxRows rows(a, seg);
      for (int j = 0; ok && j < seg.t1 - seg.t0; ++j, ++c) {
        const int st = c % STAGES, boxes = (min(PX_KEYS, seg.len - seg.start - (seg.t0 + j) * PX_KEYS) + a.box - 1) / a.box;
        ok = all_wait(empty + st * 8, ((c / STAGES) & 1) ^ 1, B2_WAIT_SMEM_EMPTY);
        if (!ok) break;
        const uint32_t bar = full + st * 8, dst = ring + st * 2 * T::TILE;
        if (b2::elect_one()) b2::mbar_arrive_expect_tx(bar, 2 * boxes * a.box * 128 * HALVES + (j == 0 ? 128 * HALVES * min(a.group, 8 * H) : 0));
        __syncwarp();
        if (j == 0) {
          if (b2::elect_one())
            for (int h = 0; h < HALVES; ++h) b2::tma_load_3d(s_q + st * T::own_q(H) + h * 1024 * H, &tmQ, bar, h * 64, seg.head * a.group + seg.row, seg.seq, b2::kEvictNormal);
          __syncwarp();
        }
        int r[4];
        rows.four(j * per_tile, r);
        if (b2::elect_one()) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < boxes)
              for (int h = 0; h < HALVES; ++h) {
                b2::tma_load_2d(dst + h * T::HALF + i * a.box * 128, &tmK, bar, seg.head * HD + h * 64, r[i], a.row_blocks > 1 ? b2::kEvictNormal : b2::kEvictFirst);
                b2::tma_load_2d(dst + T::TILE + h * T::HALF + i * a.box * 128, &tmV, bar, seg.head * HD + h * 64, r[i], a.row_blocks > 1 ? b2::kEvictNormal : b2::kEvictFirst);
              }
        }
        __syncwarp();
      }
    }
  } else {
    const int g = lane >> 2, t = lane & 3, key0 = warp * 16, swizzle = lane & 7;
    const uint32_t k_lane = (key0 + (lane & 15)) * 128, v_lane = (key0 + (lane & 7) + (lane >> 4) * 8) * 128;
    const int64_t all_rows = static_cast<int64_t>(a.n_seqs) * a.nq;
    uint32_t meetings = 0;
    auto all_here = [&]() {  // the four warps, like a barrier, but bounded
      __syncwarp();
      if (lane == 0) b2::mbar_arrive(met);
      const bool here = all_wait(met, meetings & 1, B2_WAIT_SMEM_FULL);
      ++meetings;
      return here;
    };
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      uint32_t qb[STEPS][2 * H];  // (heads behind the last one hold anything, which stays with those heads)
      float m[2 * H], l[2 * H], o[STEPS][H][4];  // heads 2 t and 2 t + 1 of each 8; dimensions g and g + 8 of each 16
#pragma unroll
      for (int h = 0; h < 2 * H; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][h][e] = 0.f;
      const int n = seg.t1 - seg.t0;
      for (int j = 0; j < n; ++j, ++c) {
        const int st = c % STAGES, there = seg.len - seg.start - (seg.t0 + j) * PX_KEYS - key0;  // keys of this warp
        ok = all_wait(full + st * 8, (c / STAGES) & 1, B2_WAIT_SMEM_FULL);
        if (!ok) break;
        __syncwarp();
        if (j == 0) {
          const uint32_t q_at = s_q + st * T::own_q(H) + (lane & (8 * H - 1)) * 128;
#pragma unroll
          for (int k = 0; k < STEPS; k += 2 / H) {
            // 16 heads: a step of 16 dimensions (heads 0 to 7, 8 to 15, the second 8 dimensions of both); 8 heads: two steps
            uint32_t r[4];
            const int chunk = (k & 3) * 2 + (H == 2 ? lane >> 4 : lane >> 3);
            b2::ldmatrix_x4(r, q_at + (k >> 2) * 1024 * H + ((chunk ^ swizzle) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) qb[H == 2 ? k : k + (e >> 1)][H == 2 ? e : e & 1] = r[e];
          }
        }
        if (there > 0) {
          const uint32_t k_at = ring + st * 2 * T::TILE + k_lane, v_at = ring + st * 2 * T::TILE + T::TILE + v_lane;
          float s[H][4] = {}, s2[H][4] = {};  // (two sums of each, so that a product waits for every other one)
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            uint32_t ka[4];
            b2::ldmatrix_x4(ka, k_at + (k >> 2) * T::HALF + (((((k & 3) * 2) + (lane >> 4)) ^ swizzle) << 4));
#pragma unroll
            for (int h = 0; h < H; ++h) mma_16x8(k & 1 ? s2[h] : s[h], ka, qb[k][h], qb[k][H + h]);
          }
          uint32_t p[H][2];
          float f[2 * H];
          bool grown = false;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            float v[4];  // key g: two heads; key g + 8
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (e >> 1) * 8 + g < there ? (s[h][e] + s2[h][e]) * a.signed_log2 : -INFINITY;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(v[e], v[2 + e]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              float &mx = m[2 * h + e], higher = fmaxf(mx, top);
              const float ref = higher == -INFINITY ? 0.f : higher;
              f[2 * h + e] = b2::ex2(mx - ref);
              grown = grown || higher > mx;
              mx = higher;
              v[e] = b2::ex2(v[e] - ref);
              v[2 + e] = b2::ex2(v[2 + e] - ref);
              l[2 * h + e] = l[2 * h + e] * f[2 * h + e] + (v[e] + v[2 + e]);
            }
            p[h][0] = transposed(b2::pack_bf16(v[0], v[1]));
            p[h][1] = transposed(b2::pack_bf16(v[2], v[3]));
          }
          if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
              for (int h = 0; h < H; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][h][e] *= f[2 * h + (e & 1)];
          }
          if (there < 16) {
            // rows of V past the context's end may hold anything, and zero times infinity or NaN is NaN: they count as zero
            for (int i = lane; i < (16 - there) * (HD / 8); i += 32) {
              const int r = there + i / (HD / 8), e = i % (HD / 8);
              *reinterpret_cast<uint4*>(smem + (v_at - v_lane - base) + (e >> 3) * T::HALF + (key0 + r) * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            uint32_t va[4];
            b2::ldmatrix_x4_trans(va, v_at + (i >> 2) * T::HALF + (((((i & 3) * 2) + ((lane >> 3) & 1)) ^ swizzle) << 4));
#pragma unroll
            for (int h = 0; h < H; ++h) mma_16x8(o[i][h], va, p[h][0], p[h][1]);
          }
        }
        __syncwarp();
        if (lane == 0) b2::mbar_arrive(empty + st * 8);
      }
      if (!ok) break;
      // ---- the warps' results together ----
#pragma unroll
      for (int h = 0; h < 2 * H; ++h) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        if (g == 0) {
          s_m[warp][(h >> 1) * 8 + 2 * t + (h & 1)] = m[h];
          s_l[warp][(h >> 1) * 8 + 2 * t + (h & 1)] = l[h];
        }
      }
      ok = all_here();
      if (!ok) break;
      auto together = [&](int r, float& top, float& sum) {
        top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < PO_WARPS; ++w) sum += s_l[w][r] * (s_m[w][r] == top ? 1.f : b2::ex2(s_m[w][r] - top));
      };
      float f[2 * H];
#pragma unroll
      for (int h = 0; h < 2 * H; ++h) {
        const int r = (h >> 1) * 8 + 2 * t + (h & 1);
        const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        f[h] = m[h] == top ? 1.f : b2::ex2(m[h] - top);
      }
      constexpr int EACH = 8 * H * DIMS / (PO_WARPS * 32);  // dimensions that a thread puts together
      const int r = tid / (DIMS / EACH), dim = tid % (DIMS / EACH) * EACH;
      float top, sum;
      together(r, top, sum);
      const bool exists = r < seg.rows, begins = seg.t0 == 0, direct = begins && seg.t1 == seg.tiles && seg.start == 0;
      const int64_t at = (static_cast<int64_t>(seg.head) * a.n_seqs + seg.seq) * a.group + seg.row + r;
      float* const slot = a.own_slots + static_cast<int64_t>(x) * T::OWN_SLOT;
#pragma unroll
      for (int d0 = 0; d0 < HD; d0 += DIMS) {
        if (d0 > 0) {  // (what was there has been read; between segments the maxima's meeting sees to that)
          ok = all_here();
          if (!ok) break;
        }
#pragma unroll
        for (int i = 0; i < DIMS / 16; ++i)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              meet[(warp * 8 * H + h * 8 + 2 * t + (e & 1)) * PAD + i * 16 + (e >> 1) * 8 + g] = o[d0 / 16 + i][h][e] * f[2 * h + (e & 1)];
        ok = all_here();
        if (!ok) break;
        if (exists) {
          float v[EACH] = {};
#pragma unroll
          for (int w = 0; w < PO_WARPS; ++w)
#pragma unroll
            for (int e = 0; e < EACH; e += 4) {
              const float4 y = *reinterpret_cast<const float4*>(meet + (w * 8 * H + r) * PAD + dim + e);
              v[e] += y.x; v[e + 1] += y.y; v[e + 2] += y.z; v[e + 3] += y.w;
            }
          if (direct) {
            const float inv = sum != 0.f ? 1.f / sum : 0.f;
            uint16_t* const to = a.out + (static_cast<int64_t>(seg.seq) * a.nq + seg.head * a.group + seg.row + r) * HD + d0 + dim;
#pragma unroll
            for (int e = 0; e < EACH; e += 4)
              *reinterpret_cast<uint2*>(to + e) = make_uint2(b2::pack_bf16(v[e] * inv, v[e + 1] * inv), b2::pack_bf16(v[e + 2] * inv, v[e + 3] * inv));
          } else {
#pragma unroll
            for (int e = 0; e < EACH; e += 4) {
              const int quad = (d0 + dim + e) / 4;
              float* const to = begins ? a.rows_o + (all_rows * HD + (quad * all_rows + at) * 4) : slot + (quad * T::OWN_ROWS + r) * 4;
              *reinterpret_cast<float4*>(to) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
          }
        }
        __syncwarp();
      }
      if (!ok) break;
      if (exists && !direct && dim == 0) {
        (begins ? a.rows_m + all_rows + at : slot + HD * T::OWN_ROWS + r)[0] = top;
        (begins ? a.rows_l + all_rows + at : slot + (HD + 1) * T::OWN_ROWS + r)[0] = sum;
      }
      __syncwarp();  // (threads that had nothing to store would go on by themselves, and what follows is for whole warps)
    }
  }
}

template <int HD, int H>
__global__ void __launch_bounds__(PX_THREADS, 1) prefix_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1, const __grid_constant__ CUtensorMap tmK,
                                                                         const __grid_constant__ CUtensorMap tmV, const PrefixArgs a) {
  using T = Prefix<HD>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const Plan plan = plan_of(reinterpret_cast<int*>(smem + T::plan(H)), a.n_groups, a.n_seqs);
  constexpr int COMMON_BARS = 2 + 4 * T::STAGES + 13, BARS = COMMON_BARS + 2 * T::OWN_STAGES + 1, P_FULL = 2 + 4 * T::STAGES + 4;
  __shared__ __align__(8) uint64_t s_bars[BARS];
  __shared__ float s_m[PO_WARPS][16], s_l[PO_WARPS][16], s_common_m[2][PX_ROWS], s_common_l[2][PX_ROWS];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t bars = b2::smem_u32(s_bars);
  const int warp = b2::uniform(static_cast<int>(threadIdx.x >> 5));
  if (threadIdx.x == 0) {
    b2::tma_prefetch_desc(&tmQ);
    b2::tma_prefetch_desc(&tmQ1);
    b2::tma_prefetch_desc(&tmK);
    b2::tma_prefetch_desc(&tmV);
    // (P by the four warps of the rows; the other keys' stages are left, and results brought together, by four warps, the common keys' results by eight)
    for (int i = 0; i < BARS; ++i) b2::mbar_init(bars + i * 8, i == COMMON_BARS - 1 ? 8 : (i >= P_FULL && i < P_FULL + 4) || i >= COMMON_BARS + T::OWN_STAGES ? 4 : 1);
    s_abort = 0;
    b2::mbar_fence_init();
  }
  if (warp == 9) {
    b2::tmem_alloc(b2::smem_u32(&s_tmem), PX_COLUMNS);
    b2::tmem_relinquish();
  }
  b2::pdl_wait();
  make_plan(a, plan, reinterpret_cast<int*>(smem));
  b2::tc_fence_before();
  __syncthreads();
  b2::tc_fence_after();
  const uint32_t tmem = b2::uniform(s_tmem);
  // (Only now: a kernel that waits for this one with columns of tensor memory in hand must not get the ones that this CTA has yet to allocate.)
  b2::pdl_launch_dependents();
  if (warp < PX_WARPS) common_keys<HD>(tmQ, tmK, tmV, a, plan, b2::smem_u32(smem), bars, tmem, s_common_m, s_common_l, warp, &s_abort);
  else own_keys<HD, H>(tmQ1, tmK, tmV, a, plan, smem, bars + COMMON_BARS * 8, s_m, s_l, warp - PX_WARPS, &s_abort);
  __syncwarp();
  b2::tc_fence_before();
  __syncthreads();
  b2::tc_fence_after();
  const int aborted = *reinterpret_cast<volatile int*>(&s_abort);
  if (aborted) {
    for (int i = 0; i < 100; ++i) __nanosleep(2000);  // copies in flight land before the CTA leaves
    if (threadIdx.x == 0) b2::report_timeout(a.status, aborted);
  }
  if (warp == 9) b2::tmem_dealloc(tmem, PX_COLUMNS);
}

// Joins the pieces of each row, in the order of their keys.  A block takes 32 rows and 64 dimensions, a thread a row and two times four dimensions.
constexpr int PJ_WARPS = 8, PJ_ROWS = 32, PJ_CTAS_PER_SM = 4;
template <int HD>
__global__ void __launch_bounds__(PJ_WARPS * 32, PJ_CTAS_PER_SM) prefix_join_kernel(const PrefixArgs a) {
  using T = Prefix<HD>;
  __shared__ __align__(16) uint16_t s_out[PJ_ROWS][64 + 8];
  __shared__ int s_store[PJ_ROWS];  // -1: stored already
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  const Plan plan = plan_of(a.plan, a.n_groups, a.n_seqs);
  const Deal common_deal(plan.common_units[a.n_groups], a.ranges), own_deal(plan.own_units[a.n_seqs], a.ranges);
  const int64_t all_rows = static_cast<int64_t>(a.n_seqs) * a.nq;
  const int blocks = static_cast<int>((all_rows + PJ_ROWS - 1) / PJ_ROWS);
  for (int u = blockIdx.x; u < blocks * (HD / 64); u += gridDim.x) {
    const int64_t at = static_cast<int64_t>(u / (HD / 64)) * PJ_ROWS + lane;
    const int dim0 = u % (HD / 64) * 64;
    bool stored = at >= all_rows;
    int to = 0;
    float top = -INFINITY, l = 0.f;
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    auto weight = [&](float m, float t) { return m == t ? 1.f : b2::ex2(m - t); };  // 1 where nothing has been seen, or for an infinity
    if (!stored) {
      const int in_head = a.n_seqs * a.group, head = static_cast<int>(at / in_head), rest = static_cast<int>(at - static_cast<int64_t>(head) * in_head), s = rest / a.group;
      to = s * a.nq + head * a.group + rest - s * a.group;
      const int g = plan.group_of[s], len = g == 0xffff ? 0 : length(a, s);
      auto add = [&](const float* p, int64_t step, float m, float sum) {
        const float t = fmaxf(top, m), f = weight(top, t), w = weight(m, t);
        l = l * f + sum * w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(dim0 / 4 + warp + 8 * k) * step);
          o[k] = make_float4(o[k].x * f + v.x * w, o[k].y * f + v.y * w, o[k].z * f + v.z * w, o[k].w * f + v.w * w);
        }
        top = t;
      };
      // the pieces of an item whose first tile is unit `first`, the row being `row` of its `rows`
      auto item = [&](int kind, const Deal& deal, int first, int tiles, const float* slots, int row, int rows) {
        const int x0 = deal.cta_of(first), x1 = deal.cta_of(first + tiles - 1);
        if (kind == 1 && x0 == x1 && plan.common_tiles(g) == 0) {  // the only piece
          stored = true;
          return;
        }
        add(a.rows_o + kind * all_rows * HD + at * 4, all_rows * 4, a.rows_m[kind * all_rows + at], a.rows_l[kind * all_rows + at]);
#pragma unroll 4
        for (int x = x0 + 1; x <= x1; ++x) {
          const float* p = slots + static_cast<int64_t>(x) * rows * (HD + 2);
          add(p + row * 4, rows * 4, p[HD * rows + row], p[(HD + 1) * rows + row]);
        }
      };
      if (len > 0) {
        const int shared = plan.common_tiles(g), j = rest - s * a.group;
        if (shared > 0) {
          const int first = bound(a, g), n = bound(a, g + 1) - first, high = (n + a.npt - 1) / a.npt, y = (s - first) / a.npt, tiles = shared;
          item(0, common_deal, plan.common_units[g] + (head * high + y) * (tiles + PX_ITEM_UNITS) + PX_ITEM_UNITS, tiles, a.slots, (s - first - y * a.npt) * a.group + j, PX_ROWS);
        }
        const int tiles = tiles_of(len - shared * PX_KEYS);
        if (tiles > 0)
          item(1, own_deal, plan.own_units[s] + (head * a.row_blocks + j / 16) * (tiles + PX_ITEM_UNITS) + PX_ITEM_UNITS, tiles, a.own_slots, j % 16, T::OWN_ROWS);
      }
    }
    // through shared memory, so that the stores are of whole pieces of rows
    const float inv = l != 0.f ? 1.f / l : 0.f;
    __syncthreads();  // (the unit before has left)
    if (warp == 0) s_store[lane] = stored ? -1 : to;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      *reinterpret_cast<uint2*>(&s_out[lane][(warp + 8 * k) * 4]) = make_uint2(b2::pack_bf16(o[k].x * inv, o[k].y * inv), b2::pack_bf16(o[k].z * inv, o[k].w * inv));
    __syncthreads();
    const int r = tid >> 3, line = s_store[r];
    if (line >= 0) *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(line) * HD + dim0 + (tid & 7) * 8) = *reinterpret_cast<const uint4*>(&s_out[r][(tid & 7) * 8]);
  }
}

struct PrefixPlan {
  int ranges, row_blocks;
  bool whole;
  int64_t rows_bytes, slots_bytes, own_bytes, bytes;
};
PrefixPlan plan_prefix(const b2_ctx* ctx, int n_seqs, int n_groups, int nq, int nkv, int head_dim, int64_t max_len) {
  PrefixPlan p;
  p.row_blocks = (nq / nkv + 15) / 16;
  const int64_t items = static_cast<int64_t>(n_seqs) * nkv * p.row_blocks;
  p.ranges = ctx->num_sms;
  // Contexts of at most PX_WHOLE_TILES tiles are not cut where there are CTAs for all of them.  (By the tables' width: the lengths are on the device.)  Not cut against cut, tables of 512 tokens that
  // come from HBM: 4 beams of 16 / 8 heads 11.6 us against 18.7, 18 of 32 / 8 heads 12.2 against 20.9, 4 of 32 / 1 heads 17.0 against 20.1, 16 of 16 / 4 heads of 64 10.3 against 17.0.  At 768 tokens
  // 13.9 / 20.3, 14.6 / 22.9, 21.0 / 21.4 and 12.0 / 18.4, at 1024 16.3 / 21.9, 17.0 / 24.6, 24.8 / 22.7 and 13.7 / 19.7: with more than eight heads a KV head the sides meet at 12 tiles, with fewer at 24.
  p.whole = max_len <= PX_WHOLE_TILES * PX_KEYS && items <= ctx->num_sms;
  if (p.whole) p.ranges = static_cast<int>(items);
  p.rows_bytes = 2ll * n_seqs * nq * (head_dim + 2) * 4;
  p.slots_bytes = static_cast<int64_t>(p.ranges) * PX_ROWS * (head_dim + 2) * 4;
  p.own_bytes = static_cast<int64_t>(p.ranges) * 16 * (head_dim + 2) * 4;
  p.bytes = p.whole ? 0 : p.rows_bytes + p.slots_bytes + p.own_bytes + (2ll * n_groups + n_seqs + 2) * 4 + (n_seqs + 1) / 2 * 4;
  return p;
}

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    constexpr auto attribute = cudaFuncAttributeMaxDynamicSharedMemorySize;
    constexpr int seqs = PX_MAX_SEQS, groups = PX_MAX_GROUPS;
    B2_CUDA((cudaFuncSetAttribute(prefix_attention_kernel<128, 1>, attribute, Prefix<128>::smem(1, seqs, groups))));
    B2_CUDA((cudaFuncSetAttribute(prefix_attention_kernel<128, 2>, attribute, Prefix<128>::smem(2, seqs, groups))));
    B2_CUDA((cudaFuncSetAttribute(prefix_attention_kernel<64, 1>, attribute, Prefix<64>::smem(1, seqs, groups))));
    B2_CUDA((cudaFuncSetAttribute(prefix_attention_kernel<64, 2>, attribute, Prefix<64>::smem(2, seqs, groups))));
    done[dev].store(true, std::memory_order_release);
  }
  return B2_OK;
}

}  // namespace

extern "C" {

int b2_prefix_attention_supported(int nq, int nkv, int head_dim, int block_size) {
  return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= PX_ROWS && nkv <= 65535 && (head_dim == 64 || head_dim == 128) && block_size > 0 && block_size % 16 == 0;
}

int64_t b2_prefix_attention_workspace(b2_ctx* ctx, int n_seqs, int n_groups, int nq, int nkv, int head_dim, int block_size, int bt_width) {
  if (ctx == nullptr || n_seqs < 0 || n_seqs > PX_MAX_SEQS || n_groups < 0 || n_groups > PX_MAX_GROUPS || bt_width < 0 ||
      !b2_prefix_attention_supported(nq, nkv, head_dim, block_size))
    return -1;
  return plan_prefix(ctx, n_seqs, n_groups, nq, nkv, head_dim, static_cast<int64_t>(bt_width) * block_size).bytes;
}

int b2_prefix_attention(b2_ctx* ctx, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int num_blocks, int block_size,
                        const int32_t* block_tables, int64_t bt_stride, int bt_width, const int32_t* cu_groups, const int32_t* prefix_lens,
                        const int32_t* context_lens, int n_groups, int max_group, int n_seqs, int nq, int nkv, int head_dim, float scale, void* out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n_seqs < 0 || n_groups < 0 || nq <= 0 || nkv <= 0 || max_group < 0) return B2_ERR_ARG;
  if (n_seqs == 0) return B2_OK;
  if (!b2_prefix_attention_supported(nq, nkv, head_dim, block_size)) return B2_ERR_UNSUPPORTED;
  if (!q || !k_cache || !v_cache || !cu_groups || !out || !block_tables || !context_lens || (n_groups > 0 && !prefix_lens)) return B2_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return B2_ERR_ARG;
  if (q_stride % 8 != 0 || q_stride < static_cast<int64_t>(nq) * head_dim || num_blocks <= 0 || bt_width <= 0 || bt_stride < bt_width) return B2_ERR_ARG;
  const int64_t max_len = static_cast<int64_t>(bt_width) * block_size;
  if (n_seqs > PX_MAX_SEQS || n_groups > PX_MAX_GROUPS) return b2::set_error(B2_ERR_SHAPE, "%d sequences, %d groups: at most %d and %d", n_seqs, n_groups, PX_MAX_SEQS, PX_MAX_GROUPS);
  // (units are counted in 32 bits)
  if (static_cast<int64_t>(num_blocks) * block_size >= 1ll << 31 || max_len >= 1ll << 27 ||
      static_cast<int64_t>(n_seqs) * nkv * ((nq / nkv + 15) / 16) * ((max_len + PX_KEYS - 1) / PX_KEYS + 2 * PX_ITEM_UNITS + 1) >= 1ll << 31 || static_cast<int64_t>(n_seqs) * nq >= 1ll << 24)
    return b2::set_error(B2_ERR_SHAPE, "%lld slots, tables of %lld tokens", static_cast<long long>(num_blocks) * block_size, static_cast<long long>(max_len));
  const PrefixPlan p = plan_prefix(ctx, n_seqs, n_groups, nq, nkv, head_dim, max_len);
  if (workspace_bytes < p.bytes || (p.bytes > 0 && workspace == nullptr)) return B2_ERR_ARG;
  const int rc = configure_once();
  if (rc != B2_OK) return rc;
  PrefixArgs a{};
  a.tables = block_tables;
  a.bt_stride = bt_stride;
  a.bt_width = bt_width;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.box = block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : 16;
  a.cu = cu_groups;
  a.prefix = prefix_lens;
  a.lens = context_lens;
  a.n_groups = n_groups;
  a.n_seqs = n_seqs;
  a.nq = nq;
  a.nkv = nkv;
  a.group = nq / nkv;
  a.npt = PX_ROWS / a.group;
  a.row_blocks = p.row_blocks;
  a.negate = scale < 0.f ? b2::kUmmaNegateA : 0u;
  a.scale_log2 = b2::scale_size(scale);
  a.signed_log2 = scale < 0.f ? -a.scale_log2 : a.scale_log2;
  a.out = static_cast<uint16_t*>(out);
  a.whole = p.whole;
  const int64_t rows = static_cast<int64_t>(n_seqs) * nq;
  a.rows_o = static_cast<float*>(workspace);
  a.rows_m = a.rows_o + 2 * rows * head_dim;
  a.rows_l = a.rows_m + 2 * rows;
  a.slots = a.rows_l + 2 * rows;
  a.own_slots = a.slots + p.slots_bytes / 4;
  a.ranges = p.ranges;
  a.plan = reinterpret_cast<int*>(a.own_slots + p.own_bytes / 4);
  a.status = ctx->status_dev;
  CUtensorMap tmQ, tmQ1, tmK, tmV;
  const uint64_t width = static_cast<uint64_t>(nkv) * head_dim, slots = static_cast<uint64_t>(num_blocks) * block_size;
  int e = b2::encode_tmap_3d(&tmQ, q, head_dim, nq, n_seqs, q_stride, 64, a.group, a.npt);
  if (e == B2_OK) e = b2::encode_tmap_3d(&tmQ1, q, head_dim, nq, n_seqs, q_stride, 64, std::min(a.group, 16), 1);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmK, k_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmV, v_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e != B2_OK) return e;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  const bool wide = head_dim == 128;
  const int h = a.group > 8 ? 2 : 1;
  const size_t smem = wide ? Prefix<128>::smem(h, n_seqs, n_groups) : Prefix<64>::smem(h, n_seqs, n_groups);
  B2_CUDA(b2_launch(wide ? (h == 2 ? prefix_attention_kernel<128, 2> : prefix_attention_kernel<128, 1>) : (h == 2 ? prefix_attention_kernel<64, 2> : prefix_attention_kernel<64, 1>), dim3(p.ranges),
                    dim3(PX_THREADS), smem, on, tmQ, tmQ1, tmK, tmV, a));
  if (!p.whole)
    B2_CUDA(b2_launch(wide ? prefix_join_kernel<128> : prefix_join_kernel<64>, dim3(PJ_CTAS_PER_SM * ctx->num_sms), dim3(PJ_WARPS * 32), 0, on, a));
  return B2_OK;
}

}  // extern "C"
