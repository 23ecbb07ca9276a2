// Decode attention over the paged KV cache for sequences that share the beginning of their contexts.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// prefix_attention_kernel
//
// Softmax over a context is the join of softmaxes over its pieces: with maxima m_k, sums l_k and unnormalised results O_k of the pieces,
// O = sum w_k O_k / sum w_k l_k, w_k = exp(m_k - max m).  So the common beginning of a group's contexts is walked once for all of its sequences, whose
// query heads fill the 128 rows of the tensor core, and the rest of each context for its own.
//
// Items are (group, KV head, 128 rows) over the common keys and (sequence, KV head) over the others, in tiles of 64 keys.  The common
// keys are those that every sequence of the group has, in whole tiles, so that no row of theirs is masked; only the last tile of a sequence is.
// The tiles of all items, first the common ones, are dealt in contiguous equal ranges to CTAs, two per SM, from lengths that are read on the device, so that a
// captured call stays balanced for any batch; CTAs that walk common keys (tensor core, exponentials) run beside those that walk others (HBM).
//
// A piece that begins an item is left in a row of its own, one for common and one for other keys, a piece that goes on with
// one that an earlier range began in the range's slot; prefix_join_kernel joins them.
//
//   warps 0..3   one thread per row: running maximum and sum, P = exp2(...) rounded to bf16 over the scores in tensor memory (the
//                product's operand has 16 bits), and the sum O rescaled where the maximum has grown
//   warp 4       TMA: Q of the segment, then K and V tiles
//   warp 5       tcgen05.mma: S = Q K^T (128 x 64, two buffers), O += P V with P read from tensor memory
// ---------------------------------------------------------------------------
constexpr int PX_ROWS = 128, PX_KEYS = 64, PX_THREADS = PX_ROWS + 64, PX_CTAS_PER_SM = 2, PX_COLUMNS = 256;
constexpr int PX_MAX_SEQS = 1024;
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
  static constexpr uint32_t PLAN = Q + 2 * STAGES * TILE;
  static constexpr size_t smem(int n_seqs, int n_groups) { return 1024 + PLAN + (2 * n_groups + n_seqs + 2) * sizeof(int) + n_seqs * sizeof(uint16_t); }
  static constexpr int SLOT = PX_ROWS * (HD + 2);  // floats of a range's piece: O as [HD / 4][row][4], then the maxima and the sums
};
static_assert(2 * (Prefix<128>::smem(PX_MAX_SEQS, PX_MAX_SEQS) + 2048) <= 228 * 1024, "two CTAs per SM (2 KB: static, reserved)");

struct PrefixArgs {
  const int32_t* tables;
  int64_t bt_stride;
  int bt_width, block_size, num_blocks, box;  // box: rows of a tensor map's box, which lie inside one block
  const int32_t *cu, *prefix, *lens;
  int n_groups, n_seqs, nq, nkv, group, npt;  // group: query heads per KV head; npt: sequences of 128 rows
  uint32_t negate;   // the instruction descriptor's bit that negates Q, where the scale is negative
  float scale_log2;  // size of softmax scale * log2(e)
  uint16_t* out;
  // pieces that begin an item: [2][HD / 4][rows][4], maxima [2][rows], sums [2][rows] for common and other keys; rows: (KV head, sequence, head of its group)
  float *rows_o, *rows_m, *rows_l;
  float* slots;     // [ranges]
  int* plan;        // for the join: units of common keys and in all, then what plan_of points into
  bool whole;       // every (sequence, KV head) is one CTA's: there are no pieces
  B2Status* status;
};

// What the batch's lengths come to, in shared memory or in the workspace.
struct Plan {
  int *common_units;  // [n_groups + 1] units of the common keys of the groups before each
  int *common;        // [n_groups] tiles of common keys, times 1024, and the sequence whose table has them
  int *own_units;     // [n_seqs + 1]
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

// Ranges of `total` units: x of X
struct Deal {
  int ctas, base, rem;
  __device__ __forceinline__ Deal(int total, int X) {
    const int per = (total + X - 1) / X;
    ctas = min(X, per <= PX_ITEM_UNITS + 6 ? (total + max(1, per) - 1) / max(1, per) : X);
    base = ctas > 0 ? total / ctas : 0;
    rem = ctas > 0 ? total % ctas : 0;
  }
  __device__ __forceinline__ int begin_of(int x) const { return x * base + min(x, rem); }
  __device__ __forceinline__ int cta_of(int t) const {
    const int big = rem * (base + 1);
    return t < big ? t / (base + 1) : rem + (t - big) / base;
  }
};

// A segment: tiles t0 .. t1 of an item with `tiles` of them, which begin at key `start` of a context of `len` keys.  rows: of the 128, from sequence seq on.
struct Segment {
  int seq, head, rows, table, start, len, tiles, t0, t1;
  bool own;
};
// A range [pos, end) of the batch's units as segments that lie inside one item.  An item has a unit for each of its tiles and, before those,
// PX_ITEM_UNITS for its beginning and its end.  A segment may hold no tiles (t0 >= t1).
struct PrefixWalk {
  const Plan plan;
  int pos, end, g, s;
  __device__ __forceinline__ static int last_at(const int* first, int n, int unit) {  // the last that begins at or before the unit
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= unit) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
  __device__ __forceinline__ PrefixWalk(const PrefixArgs& a, const Plan& p, int begin, int stop) : plan(p), pos(begin), end(stop) {
    const int common = plan.common_units[a.n_groups];
    g = last_at(plan.common_units, a.n_groups, pos);
    s = last_at(plan.own_units, a.n_seqs, max(0, pos - common));
  }
  __device__ __forceinline__ bool next(const PrefixArgs& a, Segment& x) {
    if (pos >= end) return false;
    const int common = plan.common_units[a.n_groups];
    int in_item, units;
    if (pos < common) {
      while (plan.common_units[g + 1] <= pos) ++g;
      const int first = bound(a, g), n = bound(a, g + 1) - first, high = (n + a.npt - 1) / a.npt;
      x.own = false;
      x.start = 0;
      x.tiles = plan.common_tiles(g);
      x.len = x.tiles * PX_KEYS;
      x.table = plan.leader(g);
      units = x.tiles + PX_ITEM_UNITS;
      const int in_group = pos - plan.common_units[g], item = in_group / units;
      x.head = item / high;
      const int y = item - x.head * high;
      x.seq = first + y * a.npt;
      x.rows = min(a.npt, n - y * a.npt) * a.group;
      in_item = in_group - item * units;
    } else {
      while (plan.own_units[s + 1] <= pos - common) ++s;
      x.own = true;
      x.len = length(a, s);
      x.start = plan.common_tiles(plan.group_of[s]) * PX_KEYS;
      x.table = s;
      x.tiles = tiles_of(x.len - x.start);
      units = x.tiles + PX_ITEM_UNITS;
      const int in_seq = pos - common - plan.own_units[s], item = in_seq / units;
      x.head = item;
      x.seq = s;
      x.rows = a.group;
      in_item = in_seq - item * units;
    }
    const int u1 = min(units, in_item + end - pos);
    pos += u1 - in_item;
    x.t0 = max(0, in_item - PX_ITEM_UNITS);
    x.t1 = u1 - PX_ITEM_UNITS;
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(PX_THREADS, PX_CTAS_PER_SM)
prefix_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const PrefixArgs a) {
  using T = Prefix<HD>;
  constexpr int HALVES = T::HALVES, STAGES = T::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_q = b2::smem_u32(smem), s_k = s_q + T::Q, s_v = s_k + STAGES * T::TILE;
  const Plan plan = plan_of(reinterpret_cast<int*>(smem + T::PLAN), a.n_groups, a.n_seqs);
  __shared__ __align__(8) uint64_t s_bars[2 + 4 * STAGES + 6];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  volatile int* abort_flag = &s_abort;
  const uint32_t q_full = b2::smem_u32(s_bars), q_empty = q_full + 8, k_full = q_empty + 8, k_empty = k_full + STAGES * 8, v_full = k_empty + STAGES * 8,
                 v_empty = v_full + STAGES * 8, s_full = v_empty + STAGES * 8, p_full = s_full + 2 * 8, o_done = p_full + 2 * 8;
  const int warp = b2::uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    b2::tma_prefetch_desc(&tmQ);
    b2::tma_prefetch_desc(&tmQ1);
    b2::tma_prefetch_desc(&tmK);
    b2::tma_prefetch_desc(&tmV);
    for (int i = 0; i < 2 + 4 * STAGES + 6; ++i) b2::mbar_init(q_full + i * 8, q_full + i * 8 == p_full || q_full + i * 8 == p_full + 8 ? PX_ROWS / 32 : 1);
    s_abort = 0;
    b2::mbar_fence_init();
  }
  if (warp == 5) {
    b2::tmem_alloc(b2::smem_u32(&s_tmem), PX_COLUMNS);
    b2::tmem_relinquish();
  }
  b2::pdl_wait();

  // ---- the batch's units ----
  const int X = gridDim.x, x = blockIdx.x, n_seqs = a.n_seqs, n_groups = a.n_groups;
  int* const first_live = reinterpret_cast<int*>(smem + T::Q);  // [n_groups] (where the ring will be)
  for (int g = threadIdx.x; g < n_groups; g += PX_THREADS) {
    first_live[g] = PX_MAX_SEQS;
    plan.common[g] = max(0, __ldg(a.prefix + g));
    plan.common_units[g + 1] = bound(a, g + 1);  // (for the search below)
    if (g == 0) plan.common_units[0] = bound(a, 0);
  }
  __syncthreads();
  for (int s = threadIdx.x; s < n_seqs; s += PX_THREADS) {
    const int len = length(a, s);
    int g = PrefixWalk::last_at(plan.common_units, n_groups, s);
    if (n_groups == 0 || s < plan.common_units[g] || s >= plan.common_units[g + 1]) g = 0xffff;
    plan.group_of[s] = static_cast<uint16_t>(g);
    plan.own_units[s + 1] = g == 0xffff ? 0 : len;
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
      return keys > 0 ? a.nkv * (tiles_of(keys) + PX_ITEM_UNITS) : 0;
    });
  }
  b2::tc_fence_before();
  __syncthreads();
  b2::tc_fence_after();
  const uint32_t tmem = b2::uniform(s_tmem);
  // (Only now: a kernel that waits for this one with columns of tensor memory in hand must not get the ones that this CTA has yet to allocate.)
  b2::pdl_launch_dependents();
  const int total = plan.common_units[n_groups] + plan.own_units[n_seqs];
  const Deal deal(total, X);
  int begin = x < deal.ctas ? deal.begin_of(x) : 0, end = x < deal.ctas ? deal.begin_of(x + 1) : 0;
  if (a.whole) {  // CTA x is (sequence, KV head) x
    const int s = x / a.nkv, units = (plan.own_units[s + 1] - plan.own_units[s]) / a.nkv;
    begin = plan.own_units[s] + (x - s * a.nkv) * units;
    end = begin + units;
    if (units == 0 && threadIdx.x < PX_ROWS) {  // nothing to see
      uint4* out = reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(s) * a.nq + (x - s * a.nkv) * a.group) * HD);
      for (int i = threadIdx.x; i < a.group * HD / 8; i += PX_ROWS) out[i] = make_uint4(0, 0, 0, 0);
    }
  } else if (x == 0) {
    // for the join
    const int words = 2 * n_groups + n_seqs + 2 + (n_seqs + 1) / 2;
    for (int i = threadIdx.x; i < words; i += PX_THREADS) a.plan[i] = plan.common_units[i];
  }
  PrefixWalk walk(a, plan, begin, end);
  Segment seg;
  auto all_wait = [&](uint32_t bar, uint32_t phase, int code) {
    return __all_sync(0xffffffffu, b2::mbar_wait(bar, phase, abort_flag, PX_LIMIT_NS, code)) != 0;
  };
  int c = 0, segs = 0;  // tiles and segments so far

  if (begin >= end) {
  } else if (warp == 4) {
    // ---------------- TMA (the whole warp walks and one thread issues, here and in the next warp) ----------------
    bool ok = true;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      const int32_t* table = a.tables + static_cast<int64_t>(seg.table) * a.bt_stride;
      ok = all_wait(q_empty, (segs & 1) ^ 1, B2_WAIT_SMEM_EMPTY);
      if (!ok) break;
      if (b2::elect_one()) {
        b2::mbar_arrive_expect_tx(q_full, HALVES * 128 * a.group * (seg.own ? 1 : a.npt));
        for (int i = 0; i < HALVES; ++i) b2::tma_load_3d(s_q + i * T::Q_HALF, seg.own ? &tmQ1 : &tmQ, q_full, i * 64, seg.head * a.group, seg.seq, b2::kEvictNormal);
      }
      __syncwarp();
      // Rows of the cache of 32 boxes at a time, one per lane, and those of the next 32 before they are needed: an entry of the table takes half a
      // microsecond to arrive.  K runs ahead of V, which keeps its own.
      const int per_tile = PX_KEYS / a.box, boxes_end = (seg.len + a.box - 1) / a.box, first_box = seg.start / a.box + seg.t0 * per_tile;
      auto rows_of = [&](int group) {
        const int box = first_box + group * 32 + lane, p = box * a.box, blk = p / a.block_size;
        if (box >= boxes_end) return 0;
        return min(max(0, __ldg(table + blk)), a.num_blocks - 1) * a.block_size + p - blk * a.block_size;  // inside the cache whatever the table holds
      };
      int k_rows = rows_of(0), k_next = rows_of(1), v_rows = k_rows, v_next = k_next, k_group = 0, v_group = 0;
      auto load = [&](int j, int no, const CUtensorMap* map, uint32_t full, uint32_t empty, uint32_t dst, int& rows, int& next, int& group) {
        const int st = no % STAGES, boxes = (min(PX_KEYS, seg.len - seg.start - (seg.t0 + j) * PX_KEYS) + a.box - 1) / a.box, first = j * per_tile;
        if (first >> 5 != group) {
          rows = next;
          group = first >> 5;
          next = rows_of(group + 1);
        }
        if (!all_wait(empty + st * 8, ((no / STAGES) & 1) ^ 1, B2_WAIT_SMEM_EMPTY)) return false;
        const uint32_t bar = full + st * 8;
        if (b2::elect_one()) b2::mbar_arrive_expect_tx(bar, boxes * a.box * 128 * HALVES);
        for (int i = 0; i < boxes; ++i) {
          const int r = __shfl_sync(0xffffffffu, rows, (first + i) & 31);
          if (b2::elect_one())
            for (int h = 0; h < HALVES; ++h)
              b2::tma_load_2d(dst + st * T::TILE + h * T::HALF + i * a.box * 128, map, bar, seg.head * HD + h * 64, r, seg.own ? b2::kEvictFirst : b2::kEvictNormal);
        }
        __syncwarp();
        return true;
      };
      auto load_k = [&](int j) { return load(j, c + j, &tmK, k_full, k_empty, s_k, k_rows, k_next, k_group); };
      auto load_v = [&](int j) { return load(j, c + j, &tmV, v_full, v_empty, s_v, v_rows, v_next, v_group); };
      // in the order of use: K of two tiles, then V of a tile and K of the one after the next
      const int n = seg.t1 - seg.t0;
      ok = load_k(0);
      if (n > 1) ok = ok && load_k(1);
      for (int j = 0; ok && j < n; ++j) {
        ok = load_v(j);
        if (j + 2 < n) ok = ok && load_k(j + 2);
      }
      c += n;
      ++segs;
    }
  } else if (warp == 5) {
    // ---------------- tensor core ----------------
    const uint32_t idesc_s = b2::umma_idesc_bf16(PX_KEYS) | a.negate;
    constexpr uint32_t idesc_o = b2::umma_idesc_bf16(HD) | (1u << 16);  // second operand MN-major
    const uint64_t desc_q = b2::umma_smem_desc(s_q), desc_k = b2::umma_smem_desc(s_k), desc_v = b2::umma_smem_desc_mn(s_v, T::HALF);  // (addresses in 16 bytes)
    auto wait = [&](uint32_t bar, uint32_t phase, int code) {
      const bool ok = all_wait(bar, phase, code);
      b2::tc_fence_after();
      return ok;
    };
    // scores of tile i, into the columns that P of tile i - 2 was read from, once it has been (a barrier for each of the two buffers: where a
    // segment ends, both products may be complete before this wait begins, and with one barrier it would take the later phase for one that is to come)
    auto scores = [&](int i, bool last) {
      const int st = i % STAGES;
      bool ok = i < 2 || wait(o_done + (i & 1) * 8, ((i >> 1) & 1) ^ 1, B2_WAIT_TMEM_FULL);
      ok = ok && wait(k_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL);
      if (ok && b2::elect_one()) {
        const uint64_t dk = desc_k + st * (T::TILE >> 4);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          b2::umma_bf16(tmem + (i & 1) * PX_KEYS, desc_q + (k >> 2) * (T::Q_HALF >> 4) + 2 * (k & 3), dk + (k >> 2) * (T::HALF >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
        b2::umma_commit(s_full + (i & 1) * 8);
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
      ok = wait(q_full, segs & 1, B2_WAIT_SMEM_FULL) && scores(c, n == 1);
      if (n > 1) ok = ok && scores(c + 1, n == 2);
      for (int j = 0; ok && j < n; ++j) {
        const int i = c + j, st = i % STAGES;
        ok = wait(v_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL) && wait(p_full + (i & 1) * 8, (i >> 1) & 1, B2_WAIT_TMEM_EMPTY);
        if (!ok) break;
        if (b2::elect_one()) {
          const uint64_t dv = desc_v + st * (T::TILE >> 4);
#pragma unroll
          for (int k = 0; k < PX_KEYS / 16; ++k)  // 16 tokens: 8 columns of P, 2048 bytes of V
            b2::umma_bf16_ts(tmem + 2 * PX_KEYS, tmem + (i & 1) * PX_KEYS + k * 8, dv + k * (2048 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
          b2::umma_commit(o_done + (i & 1) * 8);
          b2::umma_commit(v_empty + st * 8);
        }
        __syncwarp();
        if (j + 2 < n) ok = scores(i + 2, j + 3 == n);
      }
      c += n;
      ++segs;
    }
  } else {
    // ---------------- a thread per row ----------------
    const int row = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, t_o = tmem + 2 * PX_KEYS + lanes;
    const uint64_t scale2 = b2::pair_of(a.scale_log2, a.scale_log2);
    const int64_t all_rows = static_cast<int64_t>(n_seqs) * a.nq;
    bool ok = true;
    while (ok && walk.next(a, seg)) {
      if (seg.t0 >= seg.t1) continue;
      const int n = seg.t1 - seg.t0;
      float m = -INFINITY;  // the row's maximum, in units of scores
      uint64_t l[2] = {};   // its sum, in two pairs
      const bool idle = warp * 32 >= seg.rows;  // none of the warp's rows exists
      for (int j = 0; j < n; ++j) {
        const int i = c + j, buf = i & 1, there = seg.len - seg.start - (seg.t0 + j) * PX_KEYS;
        ok = all_wait(s_full + buf * 8, (i >> 1) & 1, B2_WAIT_TMEM_FULL);
        if (!ok) break;
        b2::tc_fence_after();
        if (there < PX_KEYS) {
          // rows of V past the context's end may hold anything, and zero times infinity or NaN is NaN: they count as zero
          const int st = i % STAGES, key = row & 63;
          ok = all_wait(v_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL);
          if (!ok) break;
          constexpr int CHUNKS = HALVES == 2 ? 8 : 4;
          unsigned char* v = smem + (s_v - s_q) + st * T::TILE + (HALVES == 2 ? (row >> 6) * T::HALF : (row >> 6) * 64) + key * 128;
          if (key >= there) {
#pragma unroll
            for (int e = 0; e < CHUNKS; ++e)  // (another piece of every row of eight, so that they do not meet in a bank)
              *reinterpret_cast<uint4*>(v + ((e ^ key) & (CHUNKS - 1)) * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (!idle) {
          const uint32_t t_s = tmem + buf * PX_KEYS + lanes;
          uint32_t r[2][32];
          b2::tmem_ld_32x32(t_s, r[0]);
          b2::tmem_ld_32x32(t_s + 32, r[1]);
          b2::tc_wait_ld(r);
          if (there < PX_KEYS) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (e >= there) r[e >> 5][e & 31] = 0xff800000u;  // -inf
          }
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
          if (j > 0 && any_grown) {
            ok = all_wait(o_done + ((i - 1) & 1) * 8, ((i - 1) >> 1) & 1, B2_WAIT_TMEM_FULL);
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
      c += n;
      ok = all_wait(o_done + ((c - 1) & 1) * 8, ((c - 1) >> 1) & 1, B2_WAIT_TMEM_FULL);
      if (!ok) break;
      b2::tc_fence_after();
      const bool direct = seg.own && seg.start == 0 && seg.t0 == 0 && seg.t1 == seg.tiles;  // the sequence's only piece
      if (!idle) {
        float sums[2];
        b2::halves_of(b2::add_pair(l[0], l[1]), sums[0], sums[1]);
        const float sum = sums[0] + sums[1], inv = sum != 0.f ? 1.f / sum : 0.f;
        const bool exists = row < seg.rows, begins = seg.t0 == 0;
        const int kind = seg.own ? 1 : 0;
        const int64_t at = (static_cast<int64_t>(seg.head) * n_seqs + seg.seq) * a.group + row;  // (sequences of 128 rows lie one after the other)
        uint16_t* out = a.out + (static_cast<int64_t>(seg.seq) * a.nq + seg.head * a.group + row) * HD;
        float* o = begins ? a.rows_o + kind * all_rows * HD + at * 4 : a.slots + static_cast<int64_t>(x) * T::SLOT + row * 4;
        const int64_t step = begins ? all_rows * 4 : PX_ROWS * 4;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t r[2][32];
          b2::tmem_ld_32x32(t_o + h * 64, r[0]);
          b2::tmem_ld_32x32(t_o + h * 64 + 32, r[1]);
          b2::tc_wait_ld(r);
          if (!exists) continue;
          if (direct) {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = b2::pack_bf16(__uint_as_float(r[g >> 2][(g & 3) * 8 + 2 * e]) * inv, __uint_as_float(r[g >> 2][(g & 3) * 8 + 2 * e + 1]) * inv);
              *reinterpret_cast<uint4*>(out + h * 64 + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int g = 0; g < 16; ++g)
              *reinterpret_cast<uint4*>(o + (h * 16 + g) * step) = make_uint4(r[g >> 3][(g & 7) * 4], r[g >> 3][(g & 7) * 4 + 1], r[g >> 3][(g & 7) * 4 + 2], r[g >> 3][(g & 7) * 4 + 3]);
          }
        }
        if (!direct && exists) {
          (begins ? a.rows_m + kind * all_rows + at : a.slots + static_cast<int64_t>(x) * T::SLOT + HD * PX_ROWS + row)[0] = m;
          (begins ? a.rows_l + kind * all_rows + at : a.slots + static_cast<int64_t>(x) * T::SLOT + (HD + 1) * PX_ROWS + row)[0] = sum;
        }
      }
      ++segs;
    }
  }

  __syncwarp();
  b2::tc_fence_before();
  __syncthreads();
  b2::tc_fence_after();
  const int aborted = *abort_flag;
  if (aborted) {
    for (int i = 0; i < 100; ++i) __nanosleep(2000);  // copies in flight land before the CTA leaves
    if (threadIdx.x == 0) b2::report_timeout(a.status, aborted);
  }
  if (warp == 5) b2::tmem_dealloc(tmem, PX_COLUMNS);
}

// Joins the pieces of each row, in the order of their keys.  A block takes 32 rows and 64 dimensions, a thread a row and two times four dimensions.
constexpr int PJ_WARPS = 8, PJ_ROWS = 32, PJ_CTAS_PER_SM = 4;
template <int HD>
__global__ void __launch_bounds__(PJ_WARPS * 32, PJ_CTAS_PER_SM) prefix_join_kernel(const PrefixArgs a, int X) {
  using T = Prefix<HD>;
  __shared__ __align__(16) uint16_t s_out[PJ_ROWS][64 + 8];
  __shared__ int s_store[PJ_ROWS];  // -1: stored already
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  const Plan plan = plan_of(a.plan, a.n_groups, a.n_seqs);
  const int common = plan.common_units[a.n_groups];
  const Deal deal(common + plan.own_units[a.n_seqs], X);
  const int64_t all_rows = static_cast<int64_t>(a.n_seqs) * a.nq;
  const int blocks = static_cast<int>((all_rows + PJ_ROWS - 1) / PJ_ROWS);
  for (int u = blockIdx.x; u < blocks * (HD / 64); u += gridDim.x) {
    const int64_t at = static_cast<int64_t>(u / (HD / 64)) * PJ_ROWS + lane;
    const int dim0 = u % (HD / 64) * 64;
    bool stored = at >= all_rows;
    int to = 0;
    float top = -INFINITY, l = 0.f;
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    auto weight = [&](float m, float t) { return m == t ? 1.f : b2::ex2((m - t) * a.scale_log2); };  // 1 where nothing has been seen, or for an infinity
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
      // the pieces of an item whose first tile is unit `first`, the row being `row` of its 128
      auto item = [&](int kind, int first, int tiles, int row) {
        const int x0 = deal.cta_of(first), x1 = deal.cta_of(first + tiles - 1);
        if (kind == 1 && x0 == x1 && plan.common_tiles(g) == 0) {  // the only piece
          stored = true;
          return;
        }
        add(a.rows_o + kind * all_rows * HD + at * 4, all_rows * 4, a.rows_m[kind * all_rows + at], a.rows_l[kind * all_rows + at]);
#pragma unroll 4
        for (int x = x0 + 1; x <= x1; ++x) {
          const float* p = a.slots + static_cast<int64_t>(x) * T::SLOT;
          add(p + row * 4, PX_ROWS * 4, p[HD * PX_ROWS + row], p[(HD + 1) * PX_ROWS + row]);
        }
      };
      if (len > 0) {
        const int shared = plan.common_tiles(g), j = rest - s * a.group;
        if (shared > 0) {
          const int first = bound(a, g), n = bound(a, g + 1) - first, high = (n + a.npt - 1) / a.npt, y = (s - first) / a.npt, tiles = shared;
          item(0, plan.common_units[g] + (head * high + y) * (tiles + PX_ITEM_UNITS) + PX_ITEM_UNITS, tiles, (s - first - y * a.npt) * a.group + j);
        }
        const int tiles = tiles_of(len - shared * PX_KEYS);
        if (tiles > 0) item(1, common + plan.own_units[s] + head * (tiles + PX_ITEM_UNITS) + PX_ITEM_UNITS, tiles, j);
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
  int x, npt;
  bool whole;
  int64_t rows_bytes, slots_bytes, bytes;
};
PrefixPlan plan_prefix(const b2_ctx* ctx, int n_seqs, int n_groups, int nq, int nkv, int head_dim, int64_t max_len) {
  PrefixPlan p;
  p.npt = PX_ROWS / (nq / nkv);
  const int64_t most = std::max<int64_t>(1, static_cast<int64_t>(n_seqs) * nkv * ((max_len + PX_KEYS - 1) / PX_KEYS + 2 * PX_ITEM_UNITS));
  p.x = static_cast<int>(std::min<int64_t>(most, ctx->num_sms * PX_CTAS_PER_SM));
  // Contexts of at most PX_WHOLE_TILES tiles are not cut where there are CTAs for all of them.  (By the tables' width: the lengths are on the device.)
  p.whole = max_len <= PX_WHOLE_TILES * PX_KEYS && n_seqs > 0 && static_cast<int64_t>(n_seqs) * nkv <= ctx->num_sms * PX_CTAS_PER_SM;
  if (p.whole) p.x = n_seqs * nkv;
  p.rows_bytes = 2ll * n_seqs * nq * (head_dim + 2) * 4;
  p.slots_bytes = static_cast<int64_t>(p.x) * PX_ROWS * (head_dim + 2) * 4;
  p.bytes = p.whole ? 0 : p.rows_bytes + p.slots_bytes + (2ll * n_groups + n_seqs + 2) * 4 + (n_seqs + 1) / 2 * 4;
  return p;
}

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    B2_CUDA(cudaFuncSetAttribute(prefix_attention_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prefix<128>::smem(PX_MAX_SEQS, PX_MAX_SEQS)));
    B2_CUDA(cudaFuncSetAttribute(prefix_attention_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prefix<64>::smem(PX_MAX_SEQS, PX_MAX_SEQS)));
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
  if (ctx == nullptr || n_seqs < 0 || n_seqs > PX_MAX_SEQS || n_groups < 0 || n_groups > PX_MAX_SEQS || bt_width < 0 ||
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
  if (n_seqs > PX_MAX_SEQS || n_groups > PX_MAX_SEQS) return b2::set_error(B2_ERR_SHAPE, "%d sequences, %d groups: at most %d", n_seqs, n_groups, PX_MAX_SEQS);
  // (units are counted in 32 bits)
  if (static_cast<int64_t>(num_blocks) * block_size >= 1ll << 31 || max_len >= 1ll << 27 ||
      static_cast<int64_t>(n_seqs) * nkv * ((max_len + PX_KEYS - 1) / PX_KEYS + 2 * PX_ITEM_UNITS + 1) >= 1ll << 31 || static_cast<int64_t>(n_seqs) * nq >= 1ll << 24)
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
  a.npt = p.npt;
  a.negate = scale < 0.f ? b2::kUmmaNegateA : 0u;
  a.scale_log2 = b2::scale_size(scale);
  a.out = static_cast<uint16_t*>(out);
  a.whole = p.whole;
  const int64_t rows = static_cast<int64_t>(n_seqs) * nq;
  a.rows_o = static_cast<float*>(workspace);
  a.rows_m = a.rows_o + 2 * rows * head_dim;
  a.rows_l = a.rows_m + 2 * rows;
  a.slots = a.rows_l + 2 * rows;
  a.plan = reinterpret_cast<int*>(a.slots + p.slots_bytes / 4);
  a.status = ctx->status_dev;
  CUtensorMap tmQ, tmQ1, tmK, tmV;
  const uint64_t width = static_cast<uint64_t>(nkv) * head_dim, slots = static_cast<uint64_t>(num_blocks) * block_size;
  int e = b2::encode_tmap_3d(&tmQ, q, head_dim, nq, n_seqs, q_stride, 64, a.group, a.npt);
  if (e == B2_OK) e = b2::encode_tmap_3d(&tmQ1, q, head_dim, nq, n_seqs, q_stride, 64, a.group, 1);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmK, k_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmV, v_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e != B2_OK) return e;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  const size_t smem = head_dim == 128 ? Prefix<128>::smem(n_seqs, n_groups) : Prefix<64>::smem(n_seqs, n_groups);
  B2_CUDA(b2_launch(head_dim == 128 ? prefix_attention_kernel<128> : prefix_attention_kernel<64>, dim3(p.x), dim3(PX_THREADS), smem, on, tmQ, tmQ1, tmK, tmV, a));
  if (!p.whole)
    B2_CUDA(b2_launch(head_dim == 128 ? prefix_join_kernel<128> : prefix_join_kernel<64>, dim3(PJ_CTAS_PER_SM * ctx->num_sms), dim3(PJ_WARPS * 32), 0, on, a, p.x));
  return B2_OK;
}

}  // extern "C"
