// Attention of trees of drafted tokens over the paged KV cache.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// tree_attention_kernel
//
// The rows of an item (sequence, KV head) are its nodes times the group's query heads, 128 of them to a tile of the tensor core
// (npt = 128 / group nodes, the heads of a node side by side); its keys are the context in tiles of 64, the tree's own nodes last.
// Every node sees all keys before the tree, so that only the one or two tiles that hold the tree look at the masks: a row's 64 bits of a tile
// are shifted out of its words and its other scores replaced by -inf.
//
// Bound: HBM for up to 128 rows (every K and V row read once: 64 keys are 32 KB, and 128 rows of products on them take half as long as
// bringing them), the softmax's units and the tensor core's operands beyond.  64 sequences of 4096 tokens with trees of 32, 32 / 8 heads (128 rows):
// 199 to 227 us by the clock; of 199 (5.5 TB/s) the walk takes 172 and the joining of the parts 13.  One of 32768 with a tree of 64, 64 / 8 heads (512 rows): 80 to 92 us by
// the clock, 0.75 to 0.86 PFLOP/s, the tensor pipe 49 % and the exponentials' 52 % busy.
//
// Work split: the tiles of the batch in the order (sequence, head, position) are dealt in contiguous equal ranges to CTAs, two per SM,
// whose lengths are read on the device, so that a captured call stays balanced for any batch.  The tiles of 128 rows of an item go to different
// CTAs that walk the same ranges (blockIdx.y), at the same time, so that HBM is read once and the others find the keys in L2.  There are as many side by side as the
// batch's longest tree needs, by max_q, and the ranges are that much fewer: sequences with smaller trees leave the CTAs of the higher tiles idle (21 ragged
// sequences, 25 nodes to a tile: 24 us where the longest tree has 25, 30 with 27, and 72 where max_q says 200 of the 27).  An item that several
// ranges share leaves its parts - unnormalised sums in 32 bits with their maxima - in the workspace, and tree_combine_kernel joins
// them in the order of the ranges.
//
//   warps 0..3   one thread per row: running maximum and sum, P = exp2(...) rounded to bf16 over the scores in tensor memory (the
//                product's operand has 16 bits), and the sum O rescaled where the maximum has grown
//   warp 4       TMA: Q of the segment, then K and V tiles
//   warp 5       tcgen05.mma: S = Q K^T (128 x 64, two buffers, so that the next tile's scores are there before this one's are done
//                with), O += P V with P read from tensor memory
// (Two threads per row, 32 keys each, which tell each other their maxima: 83 us instead of 73 for one context of 32768 tokens, tree of 64, 64 / 8 heads.)
// ---------------------------------------------------------------------------
constexpr int TR_ROWS = 128, TR_KEYS = 64, TR_THREADS = TR_ROWS + 64, TR_CTAS_PER_SM = 2, TR_COLUMNS = 256;
constexpr int TR_MAX_SEQS = 1024;
constexpr int TR_ITEM_UNITS = 2;   // what an item costs beside its tiles, in tiles (21 ragged sequences, the longest CTA 32 us without them, 26 with)
// Contexts whole and cut (tables as narrow as they can be, 16 / 8 heads, trees of 5; one sequence: 8 items, eight: 64): 4 tiles 9.3 and 10.1 us, 10.1 and 14.8;
// 6 tiles 11.0 and 11.0, 11.8 and 15.1; 8 tiles 12.6 and 11.1, 13.5 and 16.3; 12 tiles 15.9 and 11.7, 16.9 and 17.5.  The line lies at 6 tiles for one sequence and behind 12
// for eight; 8 gives away an eighth of the one to win a sixth of the other.
constexpr int TR_WHOLE_TILES = 8;
constexpr float TR_GROWTH = 8.f;
constexpr uint64_t TR_LIMIT_NS = 1000000000ull;
template <int HD>
struct Tree {
  static constexpr int HALVES = HD / 64;
  static constexpr int STAGES = 4 / HALVES;                 // tiles of K, and as many of V
  static constexpr uint32_t HALF = TR_KEYS * 128;           // 64 keys of 64 dimensions: one swizzled box
  static constexpr uint32_t TILE = HALVES * HALF;
  static constexpr uint32_t Q_HALF = TR_ROWS * 128;
  static constexpr uint32_t Q = HALVES * Q_HALF;
  static constexpr size_t smem(int n_seqs) { return 1024 + Q + 2 * STAGES * TILE + (n_seqs + 1) * sizeof(int); }
  static constexpr int SLOT = TR_ROWS * (HD + 2);           // floats of a part: O as [HD / 4][row][4], then the maxima and the sums
};
static_assert(2 * (Tree<128>::smem(TR_MAX_SEQS) + 2048) <= 228 * 1024, "two CTAs per SM (2 KB: static, reserved)");

struct TreeArgs {
  const uint16_t* v;
  const int32_t* tables;
  int64_t bt_stride;
  int bt_width, block_size, num_blocks, box;  // box: rows of a tensor map's box, which lie inside one block
  const int32_t *cu_q, *lens;
  const int64_t* mask;
  int64_t mask_stride;
  int words, n_seqs, tokens, nq, nkv, group, npt;
  uint32_t negate;   // the instruction descriptor's bit that negates Q, where the scale is negative
  float scale_log2;  // size of softmax scale * log2(e)
  uint16_t* out;
  float* parts;      // [2][gridDim.y][gridDim.x] slots: [0] of the item that a range begins in, [1] of the one it ends in
  bool whole;        // every (sequence, KV head) is one CTA's: there are no parts
  int4* joins;       // [gridDim.y][gridDim.x]: parts of the item that the range ends in (0: none), its first token, its nodes in the tile, its KV head
  B2Status* status;
};

struct Sequence {
  int q0, nodes, len;
};
// Nodes and context of a sequence, and no tiles for one whose context is shorter than its tree.
__device__ __forceinline__ Sequence sequence(const TreeArgs& a, int b) {
  const int q0 = __ldg(a.cu_q + b), nodes = __ldg(a.cu_q + b + 1) - q0;
  const int len = min(__ldg(a.lens + b), a.bt_width * a.block_size);
  return {q0, nodes, q0 >= 0 && nodes > 0 && q0 + nodes <= a.tokens && len >= nodes ? len : 0};
}
__device__ __forceinline__ int tiles_of(int len) { return (len + TR_KEYS - 1) / TR_KEYS; }

// A range [pos, end) of the batch's units as segments that lie inside one item.  An item has a unit for each of its tiles and, before those,
// TR_ITEM_UNITS for its beginning and its end (loading Q, the tree's masks, storing O).  A sequence with more nodes than gridDim.y tiles of rows hold
// is walked several times (pass).  A segment may hold no tiles (t0 >= t1).
struct TreeWalk {
  const int* first_unit_of;  // [n_seqs + 1] units per KV head before each sequence
  int nkv, pos, end, jump, again, b, head, pass, tiles, t0, t1;
  // again: so many further ranges of the same length, `jump` units behind the end of the one before
  __device__ __forceinline__ TreeWalk(const int* fu, int n_seqs, int heads, int begin, int stop, int jump, int again)
      : first_unit_of(fu), nkv(heads), pos(begin), end(stop), jump(jump), again(again), b(0) {
    int hi = n_seqs - 1;
    while (b < hi) {
      const int mid = (b + hi + 1) >> 1;
      if (first_unit_of[mid] * nkv <= pos) b = mid;
      else hi = mid - 1;
    }
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, Sequence& s) {
    if (pos >= end) {
      if (--again < 0) return false;
      const int units = tiles + TR_ITEM_UNITS;
      pos += jump;
      end = pos + units;
    }
    while (first_unit_of[b + 1] * nkv <= pos) ++b;
    s = sequence(a, b);
    tiles = tiles_of(s.len);
    const int units = tiles + TR_ITEM_UNITS, in_seq = pos - first_unit_of[b] * nkv, item = in_seq / units;
    pass = item / nkv;
    head = item - pass * nkv;
    const int u0 = in_seq - item * units, u1 = min(units, u0 + end - pos);
    pos += u1 - u0;
    t0 = max(0, u0 - TR_ITEM_UNITS);
    t1 = u1 - TR_ITEM_UNITS;
    return true;
  }
  // the unit of the item's first tile, after a segment that holds some
  __device__ __forceinline__ int first_unit() const { return pos - t1; }
};

// Bits 64 tile .. of what row `words` of the mask sees, for a tile that begins `off` places after the tree does (before it: negative)
__device__ __forceinline__ uint64_t visible(const int64_t* row, int words, int off) {
  auto word = [&](int w) { return w < words ? __ldg(reinterpret_cast<const unsigned long long*>(row) + w) : 0ull; };
  if (off < 0) return (word(0) << -off) | ((1ull << -off) - 1);  // (off > -64)
  const int w = off >> 6, s = off & 63;
  return s == 0 ? word(w) : (word(w) >> s) | (word(w + 1) << (64 - s));
}

// What infinities and NaN in the values (one element of each) of the tree's nodes from place p0 to p1 add to a row that sees some of them.  They
// are zero in shared memory, where they would reach every row: zero times them is NaN.
__device__ __noinline__ float unbounded(const uint16_t* v, int64_t v_row, const int32_t* table, int block_size, int num_blocks, const int64_t* row, int words,
                                        int prefix, int p0, int p1) {
  float sum = 0.f;
  for (int p = max(p0, prefix); p < p1; ++p) {
    const int node = p - prefix, no = p / block_size;
    if (node >= 64 * words || !((__ldg(reinterpret_cast<const unsigned long long*>(row) + (node >> 6)) >> (node & 63)) & 1)) continue;
    const int block = min(max(0, __ldg(table + no)), num_blocks - 1);
    const uint16_t x = v[(static_cast<int64_t>(block) * block_size + (p - no * block_size)) * v_row];
    if ((x & 0x7f80u) == 0x7f80u) sum += b2::bf16_lo(x);
  }
  return sum;
}

__device__ __forceinline__ bool any_unbounded(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t without_unbounded(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

template <int HD>
__global__ void __launch_bounds__(TR_THREADS, TR_CTAS_PER_SM)
tree_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeArgs a) {
  using T = Tree<HD>;
  constexpr int HALVES = T::HALVES, STAGES = T::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_q = b2::smem_u32(smem), s_k = s_q + T::Q, s_v = s_k + STAGES * T::TILE;
  int* first_unit = reinterpret_cast<int*>(smem + T::Q + 2 * STAGES * T::TILE);
  __shared__ __align__(8) uint64_t s_bars[2 + 4 * STAGES + 6];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_unbounded[2];
  volatile int* abort_flag = &s_abort;
  const uint32_t q_full = b2::smem_u32(s_bars), q_empty = q_full + 8, k_full = q_empty + 8, k_empty = k_full + STAGES * 8, v_full = k_empty + STAGES * 8,
                 v_empty = v_full + STAGES * 8, s_full = v_empty + STAGES * 8, p_full = s_full + 2 * 8, o_done = p_full + 2 * 8;
  const int warp = b2::uniform(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    b2::tma_prefetch_desc(&tmQ);
    b2::tma_prefetch_desc(&tmK);
    b2::tma_prefetch_desc(&tmV);
    for (int i = 0; i < 2 + 4 * STAGES + 6; ++i) b2::mbar_init(q_full + i * 8, q_full + i * 8 == p_full || q_full + i * 8 == p_full + 8 ? TR_ROWS / 32 : 1);
    s_abort = 0;
    s_unbounded[0] = s_unbounded[1] = -1;
    b2::mbar_fence_init();
  }
  if (warp == 5) {
    b2::tmem_alloc(b2::smem_u32(&s_tmem), TR_COLUMNS);
    b2::tmem_relinquish();
  }
  b2::pdl_wait();

  // ---- units per sequence, prefix-summed by one warp ----
  const int X = gridDim.x, Y = gridDim.y, rows_y = Y * a.npt;
  if (warp == 0) {
    const int per = (a.n_seqs + 31) / 32, s0 = lane * per;
    int mine = 0;
#pragma unroll 4
    for (int i = 0; i < per; ++i)
      if (s0 + i < a.n_seqs) {
        const Sequence s = sequence(a, s0 + i);
        const int all = s.len > 0 ? (tiles_of(s.len) + TR_ITEM_UNITS) * ((s.nodes + rows_y - 1) / rows_y) : 0;
        first_unit[s0 + i + 1] = all;
        mine += all;
      }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    int at = incl - mine;
    if (lane == 0) first_unit[0] = 0;
    for (int i = 0; i < per; ++i)
      if (s0 + i < a.n_seqs) first_unit[s0 + i + 1] = at += first_unit[s0 + i + 1];
  }
  b2::tc_fence_before();
  __syncthreads();
  b2::tc_fence_after();
  const uint32_t tmem = b2::uniform(s_tmem);
  // (Only now: a kernel that waits for this one with columns of tensor memory in hand must not get the ones that this CTA has yet to allocate.)
  b2::pdl_launch_dependents();
  const int x = blockIdx.x, y = blockIdx.y, total = first_unit[a.n_seqs] * a.nkv;

  // ---- rows without anything to see: of sequences with a context shorter than their tree, and behind the last sequence (by the warps of the
  // rows, while the first tiles are on their way) ----
  auto clear_rows = [&]() {
    const int row = a.nq * HD / 8, cta = y * X + x, ctas = X * Y;
    auto clear = [&](int from, int to) {
      from = max(from, 0);
      uint4* out = reinterpret_cast<uint4*>(a.out) + static_cast<int64_t>(from) * row;
      const int64_t n = static_cast<int64_t>(min(to, a.tokens) - from) * row;
      for (int64_t i = threadIdx.x; i < n; i += TR_ROWS) out[i] = make_uint4(0, 0, 0, 0);
    };
    for (int b = cta; b < a.n_seqs; b += ctas) {
      const Sequence s = sequence(a, b);
      if (s.len == 0) clear(s.q0, s.q0 + s.nodes);
    }
    if (cta == 0 && a.n_seqs > 0) clear(0, __ldg(a.cu_q));
    const int behind = a.n_seqs > 0 ? max(0, __ldg(a.cu_q + a.n_seqs)) : 0;
    for (int t = behind + cta; t < a.tokens; t += ctas) clear(t, t + 1);
  };

  // ---- this CTA's range ----
  const int per = (total + X - 1) / X;
  const int ctas = min(X, per <= TR_ITEM_UNITS + 6 ? (total + max(1, per) - 1) / max(1, per) : X);
  const int base = ctas > 0 ? total / ctas : 0, rem = ctas > 0 ? total % ctas : 0;
  auto begin_of = [&](int i) { return i * base + min(i, rem); };
  auto cta_of = [&](int t) { const int big = rem * (base + 1); return t < big ? t / (base + 1) : rem + (t - big) / base; };
  int begin = x < ctas ? begin_of(x) : 0, end = x < ctas ? begin_of(x + 1) : 0, jump = 0, again = 0;
  Sequence s;
  if (a.whole) {  // CTA x is (sequence, KV head) x: one range, or one for each pass
    const int b = x / a.nkv;
    s = sequence(a, b);
    const int units = tiles_of(s.len) + TR_ITEM_UNITS;
    begin = first_unit[b] * a.nkv + (x - b * a.nkv) * units;
    end = s.len > 0 ? begin + units : begin;
    jump = (a.nkv - 1) * units;
    again = (first_unit[b + 1] - first_unit[b]) / units - 1;
  }
  TreeWalk walk(first_unit, a.n_seqs, a.nkv, begin, end, jump, again);
  auto all_wait = [&](uint32_t bar, uint32_t phase, int code) {
    return __all_sync(0xffffffffu, b2::mbar_wait(bar, phase, abort_flag, TR_LIMIT_NS, code)) != 0;
  };
  // the nodes of this CTA's tile of rows: first, number
  auto first_node = [&]() { return (walk.pass * Y + y) * a.npt; };
  int c = 0, seg = 0;  // tiles and segments so far

  if (begin >= end) {
    if (warp < 4) clear_rows();
    if (threadIdx.x == 0 && !a.whole) a.joins[y * X + x] = make_int4(0, 0, 0, 0);
  } else if (warp == 4) {
    // ---------------- TMA (the whole warp walks and one thread issues, here and in the next warp) ----------------
    bool ok = true;
    while (ok && walk.next(a, s)) {
      const int n0 = first_node();
      if (n0 >= s.nodes || walk.t0 >= walk.t1) continue;
      const int32_t* table = a.tables + static_cast<int64_t>(walk.b) * a.bt_stride;
      ok = all_wait(q_empty, (seg & 1) ^ 1, B2_WAIT_SMEM_EMPTY);
      if (!ok) break;
      if (b2::elect_one()) {
        b2::mbar_arrive_expect_tx(q_full, HALVES * 128 * a.npt * a.group);
        for (int i = 0; i < HALVES; ++i) b2::tma_load_3d(s_q + i * T::Q_HALF, &tmQ, q_full, i * 64, walk.head * a.group, s.q0 + n0, b2::kEvictNormal);
      }
      __syncwarp();
      // Rows of the cache of 32 boxes at a time, one per lane, and those of the next 32 before they are needed: an entry of the table takes half a
      // microsecond to arrive.  Tile j of the segment's first is in boxes j * per_tile ...; K runs ahead of V, which keeps its own.
      const int per_tile = TR_KEYS / a.box, boxes_end = (s.len + a.box - 1) / a.box;
      auto rows_of = [&](int group) {
        const int box = walk.t0 * per_tile + group * 32 + lane, p = box * a.box, blk = p / a.block_size;
        if (box >= boxes_end) return 0;
        return min(max(0, __ldg(table + blk)), a.num_blocks - 1) * a.block_size + p - blk * a.block_size;  // inside the cache whatever the table holds
      };
      int k_rows = rows_of(0), k_next = rows_of(1), v_rows = k_rows, v_next = k_next, k_group = 0, v_group = 0;
      auto load = [&](int j, int no, const CUtensorMap* map, uint32_t full, uint32_t empty, uint32_t dst, int& rows, int& next, int& group) {
        const int st = no % STAGES, boxes = (min(TR_KEYS, s.len - (walk.t0 + j) * TR_KEYS) + a.box - 1) / a.box, first = j * per_tile;
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
              b2::tma_load_2d(dst + st * T::TILE + h * T::HALF + i * a.box * 128, map, bar, walk.head * HD + h * 64, r, Y > 1 ? b2::kEvictNormal : b2::kEvictFirst);
        }
        __syncwarp();
        return true;
      };
      auto load_k = [&](int j) { return load(j, c + j, &tmK, k_full, k_empty, s_k, k_rows, k_next, k_group); };
      auto load_v = [&](int j) { return load(j, c + j, &tmV, v_full, v_empty, s_v, v_rows, v_next, v_group); };
      // in the order of use: K of two tiles, then V of a tile and K of the one after the next
      const int n = walk.t1 - walk.t0;
      ok = load_k(0);
      if (n > 1) ok = ok && load_k(1);
      for (int j = 0; ok && j < n; ++j) {
        ok = load_v(j);
        if (j + 2 < n) ok = ok && load_k(j + 2);
      }
      c += n;
      ++seg;
    }
  } else if (warp == 5) {
    // ---------------- tensor core ----------------
    const uint32_t idesc_s = b2::umma_idesc_bf16(TR_KEYS) | a.negate;
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
          b2::umma_bf16(tmem + (i & 1) * TR_KEYS, desc_q + (k >> 2) * (T::Q_HALF >> 4) + 2 * (k & 3), dk + (k >> 2) * (T::HALF >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
        b2::umma_commit(s_full + (i & 1) * 8);
        b2::umma_commit(k_empty + st * 8);
        if (last) b2::umma_commit(q_empty);
      }
      __syncwarp();
      return ok;
    };
    bool ok = true;
    while (ok && walk.next(a, s)) {
      if (first_node() >= s.nodes || walk.t0 >= walk.t1) continue;
      const int n = walk.t1 - walk.t0;
      ok = wait(q_full, seg & 1, B2_WAIT_SMEM_FULL) && scores(c, n == 1);
      if (n > 1) ok = ok && scores(c + 1, n == 2);
      for (int j = 0; ok && j < n; ++j) {
        const int i = c + j, st = i % STAGES;
        ok = wait(v_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL) && wait(p_full + (i & 1) * 8, (i >> 1) & 1, B2_WAIT_TMEM_EMPTY);
        if (!ok) break;
        if (b2::elect_one()) {
          const uint64_t dv = desc_v + st * (T::TILE >> 4);
#pragma unroll
          for (int k = 0; k < TR_KEYS / 16; ++k)  // 16 tokens: 8 columns of P, 2048 bytes of V
            b2::umma_bf16_ts(tmem + 2 * TR_KEYS, tmem + (i & 1) * TR_KEYS + k * 8, dv + k * (2048 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
          b2::umma_commit(o_done + (i & 1) * 8);
          b2::umma_commit(v_empty + st * 8);
        }
        __syncwarp();
        if (j + 2 < n) ok = scores(i + 2, j + 3 == n);
      }
      c += n;
      ++seg;
    }
  } else if (warp < 4) {
    // ---------------- a thread per row ----------------
    const int row = threadIdx.x, my_node = row / a.group, my_head = row - my_node * a.group;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, t_o = tmem + 2 * TR_KEYS + lanes;
    const uint64_t scale2 = b2::pair_of(a.scale_log2, a.scale_log2);
    bool ok = true;
    int4 join = make_int4(0, 0, 0, 0);
    clear_rows();
    while (ok && walk.next(a, s)) {
      const int n0 = first_node(), nodes = min(a.npt, s.nodes - n0), prefix = s.len - s.nodes;
      if (nodes <= 0 || walk.t0 >= walk.t1) continue;
      const int n = walk.t1 - walk.t0;
      const int token = s.q0 + n0 + min(my_node, nodes - 1);  // (rows behind the last node go along with it)
      const int64_t* mask = a.mask + static_cast<int64_t>(token) * a.mask_stride;
      float m = -INFINITY;  // the row's maximum, in units of scores
      uint64_t l[2] = {};   // its sum, in two pairs
      const bool idle = warp * 32 >= nodes * a.group;  // none of the warp's rows exists
      for (int j = 0; j < n; ++j) {
        const int i = c + j, buf = i & 1, place = (walk.t0 + j) * TR_KEYS, off = place - prefix, there = s.len - place;
        const bool special = off > -TR_KEYS || there < TR_KEYS;
        uint64_t sees = off > -TR_KEYS ? visible(mask, a.words, off) : ~0ull;  // (on its way while the scores are)
        if (there < TR_KEYS) sees &= (1ull << there) - 1;
        ok = all_wait(s_full + buf * 8, (i >> 1) & 1, B2_WAIT_TMEM_FULL);
        if (!ok) break;
        b2::tc_fence_after();
        if (special) {
          // Rows of V past the context's end count as zero, and so do infinities and NaN in the tree's: a row that does not see them
          // has a probability of zero there, and zero times them is NaN.
          const int st = i % STAGES, key = row & 63;
          ok = all_wait(v_full + st * 8, (i / STAGES) & 1, B2_WAIT_SMEM_FULL);
          if (!ok) break;
          constexpr int CHUNKS = HALVES == 2 ? 8 : 4;
          unsigned char* v = smem + (s_v - s_q) + st * T::TILE + (HALVES == 2 ? (row >> 6) * T::HALF : (row >> 6) * 64) + key * 128;
          if (key >= there) {
#pragma unroll
            for (int e = 0; e < CHUNKS; ++e)  // (another piece of every row of eight, so that they do not meet in a bank)
              *reinterpret_cast<uint4*>(v + ((e ^ key) & (CHUNKS - 1)) * 16) = make_uint4(0, 0, 0, 0);
          } else if (off + key >= 0) {
#pragma unroll
            for (int e = 0; e < CHUNKS; ++e) {
              uint4* p = reinterpret_cast<uint4*>(v + ((e ^ key) & (CHUNKS - 1)) * 16);
              const uint4 w = *p;
              if (any_unbounded(w.x) || any_unbounded(w.y) || any_unbounded(w.z) || any_unbounded(w.w)) {
                *p = make_uint4(without_unbounded(w.x), without_unbounded(w.y), without_unbounded(w.z), without_unbounded(w.w));
                s_unbounded[seg & 1] = seg;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (!idle) {
          const uint32_t t_s = tmem + buf * TR_KEYS + lanes;
          uint32_t r[2][32];
          b2::tmem_ld_32x32(t_s, r[0]);
          b2::tmem_ld_32x32(t_s + 32, r[1]);
          b2::tc_wait_ld(r);
          if (special) {
            const uint32_t half[2] = {static_cast<uint32_t>(sees), static_cast<uint32_t>(sees >> 32)};
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (!((half[e >> 5] >> (e & 31)) & 1)) r[e >> 5][e & 31] = 0xff800000u;  // -inf
          }
          float mx[4] = {m, m, m, m};
#pragma unroll
          for (int e = 0; e < 64; e += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], __uint_as_float(r[e >> 5][(e & 31) + k]));
          // The reference m moves when the row is TR_GROWTH past it (or has seen its first key): O then has to be rescaled, which takes as long as
          // half a tile.  Until then probabilities are up to 2^TR_GROWTH and rounded relative to themselves, the largest one too, which would be exactly one
          // at a reference that is the maximum.  What that costs, as the norm of the error over the norm (64 / 8 heads, a tree of 64 behind 8192 tokens, queries
          // of size 0.3 / 1 / 2): 2.32e-3 / 2.32e-3 / 2.26e-3, with every growth taken up at once 2.31e-3 / 2.21e-3 / 1.81e-3 (1.66e-3 is the result's own rounding);
          // what it saves: 77 instead of 88 us for one context of 32768, 199 instead of 204 for 64 of 4096.
          // (Each row for itself: its result does not depend on the rows beside it.)
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool grown = (top - m) * a.scale_log2 > TR_GROWTH;
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
      const bool whole = walk.t0 == 0 && walk.t1 == walk.tiles;
      if (!idle) {
        float sums[2];
        b2::halves_of(b2::add_pair(l[0], l[1]), sums[0], sums[1]);
        const float sum = sums[0] + sums[1], inv = sum != 0.f ? 1.f / sum : 0.f;  // (nothing seen: zeros)
        const bool exists = my_node < nodes;
        const bool add = *reinterpret_cast<volatile int*>(&s_unbounded[seg & 1]) == seg;
        const int32_t* table = a.tables + static_cast<int64_t>(walk.b) * a.bt_stride;
        const int p0 = walk.t0 * TR_KEYS, p1 = min(s.len, walk.t1 * TR_KEYS);
        uint16_t* out = a.out + (static_cast<int64_t>(token) * a.nq + walk.head * a.group + my_head) * HD;
        float* slot = a.parts + (static_cast<int64_t>(walk.t0 == 0 ? 1 : 0) * Y * X + y * X + x) * T::SLOT;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t r[2][32];
          b2::tmem_ld_32x32(t_o + h * 64, r[0]);
          b2::tmem_ld_32x32(t_o + h * 64 + 32, r[1]);
          b2::tc_wait_ld(r);
          if (add) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              r[e >> 5][e & 31] = __float_as_uint(__uint_as_float(r[e >> 5][e & 31]) + unbounded(a.v + walk.head * HD + h * 64 + e, static_cast<int64_t>(a.nkv) * HD, table, a.block_size,
                                                                                                                a.num_blocks, mask, a.words, prefix, p0, p1));
          }
          if (!exists) continue;
          if (whole) {
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
              *reinterpret_cast<uint4*>(slot + ((h * 16 + g) * TR_ROWS + row) * 4) =
                  make_uint4(r[g >> 3][(g & 7) * 4], r[g >> 3][(g & 7) * 4 + 1], r[g >> 3][(g & 7) * 4 + 2], r[g >> 3][(g & 7) * 4 + 3]);
          }
        }
        if (!whole && exists) {
          slot[HD * TR_ROWS + row] = m;
          slot[(HD + 1) * TR_ROWS + row] = sum;
        }
      }
      if (walk.t0 == 0 && walk.t1 < walk.tiles) {
        const int first = walk.first_unit();
        join = make_int4(cta_of(first + walk.tiles - 1) - cta_of(first) + 1, s.q0 + n0, nodes, walk.head);
      }
      ++seg;
    }
    if (threadIdx.x == 0 && !a.whole) a.joins[y * X + x] = join;
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
  if (warp == 5) b2::tmem_dealloc(tmem, TR_COLUMNS);
}

// Joins the parts of the items that several ranges share: O = sum w O_k / sum w l_k with w = exp2(m_k - max m), the parts in the order of
// their keys.  Few parts: a block takes 32 rows and 64 dimensions of an item, every thread all parts of its elements.  Many: 32 rows and 16 dimensions,
// its warps every eighth part each, which then meet in shared memory.  (64 sequences of 4096 tokens, 128 rows, 2 to 3 parts an item: 60 us where the
// warps always shared the parts, of which most had none.)
constexpr int TC_WARPS = 8, TC_ROWS = 32, TC_FEW = 16, TC_CTAS_PER_SM = 4;
template <int HD>
__global__ void __launch_bounds__(TC_WARPS * 32, TC_CTAS_PER_SM) tree_combine_kernel(const TreeArgs a, int X, int Y) {
  using T = Tree<HD>;
  __shared__ int s_units[TC_WARPS * 32 + 1], s_sum[TC_WARPS];
  __shared__ float s_m[TC_WARPS][TC_ROWS], s_l[TC_WARPS][TC_ROWS];
  __shared__ float4 s_o[TC_WARPS][4][TC_ROWS];
  __shared__ int4 s_join[TC_WARPS * 32];
  __shared__ __align__(16) uint16_t s_out[TC_ROWS][64 + 8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = X * Y;
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  // units of all items, prefix-summed in chunks of a block's threads (there are one or two)
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += TC_WARPS * 32) {
    const int4 mine = i0 + tid < n ? a.joins[i0 + tid] : make_int4(0, 0, 0, 0);
    const int units = mine.x > 0 ? (mine.z * a.group + TC_ROWS - 1) / TC_ROWS * (HD / (mine.x <= TC_FEW ? 64 : 16)) : 0;
    int incl = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < warp; ++w) at += s_sum[w];
    s_units[tid] = at + incl - units;
    s_join[tid] = mine;
    if (tid == TC_WARPS * 32 - 1) s_units[TC_WARPS * 32] = at + incl;
    __syncthreads();
    const int all = s_units[TC_WARPS * 32];
    int u = static_cast<int>(blockIdx.x) - before % static_cast<int>(gridDim.x);
    if (u < 0) u += gridDim.x;
    for (; u < all; u += gridDim.x) {
      int lo = 0, hi = TC_WARPS * 32 - 1;  // the last entry that begins at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_units[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      const int e = i0 + lo, part = u - s_units[lo];
      const int4 join = s_join[lo];
      const int parts = join.x;
      // the item begins in range e (its slot [1]) and goes on in the ranges after it (their slots [0])
      auto slot = [&](int k) { return a.parts + (k == 0 ? static_cast<int64_t>(Y) * X + e : static_cast<int64_t>(e) + k) * T::SLOT; };
      auto store = [&](int row, int dim, const float4& o, float l) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const int token = join.y + row / a.group, head = join.w * a.group + row % a.group;
        *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(token) * a.nq + head) * HD + dim) = make_uint2(b2::pack_bf16(o.x * inv, o.y * inv), b2::pack_bf16(o.z * inv, o.w * inv));
      };
      auto add = [](float4& acc, float f, const float4& o) { acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w; };
      // 0 for a part that saw nothing where another one did; 1 where none did, or for an infinity
      auto weight = [&](float m, float top) { return m == top ? 1.f : b2::ex2((m - top) * a.scale_log2); };
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      if (parts <= TC_FEW) {
        const int row = part / (HD / 64) * TC_ROWS + lane, quad = part % (HD / 64) * 16 + warp;
        const int rows = join.z * a.group;
        float top = -INFINITY, l = 0.f;
        float4 o0 = zero, o1 = zero;
        for (int k0 = 0; row < rows && k0 < parts; k0 += 4) {  // four parts at a time, all of them on their way at once
          float m[4], sums[4];
          float4 u[4], w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            m[k] = -INFINITY;
            sums[k] = 0.f;
            u[k] = w[k] = zero;
            if (k0 + k < parts) {
              const float* p = slot(k0 + k);
              m[k] = p[HD * TR_ROWS + row];
              sums[k] = p[(HD + 1) * TR_ROWS + row];
              u[k] = *reinterpret_cast<const float4*>(p + (quad * TR_ROWS + row) * 4);
              w[k] = *reinterpret_cast<const float4*>(p + ((quad + 8) * TR_ROWS + row) * 4);
            }
          }
          const float before = top;
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, m[k]);
          const float g = weight(before, top);
          l *= g;
          o0.x *= g; o0.y *= g; o0.z *= g; o0.w *= g;
          o1.x *= g; o1.y *= g; o1.z *= g; o1.w *= g;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float f = weight(m[k], top);
            l += f * sums[k];
            add(o0, f, u[k]);
            add(o1, f, w[k]);
          }
        }
        // through shared memory, so that the stores are of whole pieces of rows
        const float inv = l != 0.f ? 1.f / l : 0.f;
        __syncthreads();  // (the unit before has left)
        *reinterpret_cast<uint2*>(&s_out[lane][warp * 4]) = make_uint2(b2::pack_bf16(o0.x * inv, o0.y * inv), b2::pack_bf16(o0.z * inv, o0.w * inv));
        *reinterpret_cast<uint2*>(&s_out[lane][warp * 4 + 32]) = make_uint2(b2::pack_bf16(o1.x * inv, o1.y * inv), b2::pack_bf16(o1.z * inv, o1.w * inv));
        __syncthreads();
        const int r = row - lane + (tid >> 3);
        if (r < rows)
          *reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(join.y + r / a.group) * a.nq + join.w * a.group + r % a.group) * HD + part % (HD / 64) * 64 + (tid & 7) * 8) =
              *reinterpret_cast<const uint4*>(&s_out[tid >> 3][(tid & 7) * 8]);
        continue;
      }
      const int row = part / (HD / 16) * TC_ROWS + lane, quad = part % (HD / 16) * 4;
      const bool exists = row < join.z * a.group;
      float mx = -INFINITY, sum = 0.f;
      float4 acc[4] = {zero, zero, zero, zero};
      if (exists) {
        for (int k = warp; k < parts; k += TC_WARPS) mx = fmaxf(mx, slot(k)[HD * TR_ROWS + row]);
#pragma unroll 2
        for (int k = warp; k < parts; k += TC_WARPS) {
          const float* p = slot(k);
          const float f = weight(p[HD * TR_ROWS + row], mx);
          sum += f * p[(HD + 1) * TR_ROWS + row];
#pragma unroll
          for (int d = 0; d < 4; ++d) add(acc[d], f, *reinterpret_cast<const float4*>(p + ((quad + d) * TR_ROWS + row) * 4));
        }
      }
      __syncthreads();
      s_m[warp][lane] = mx;
      s_l[warp][lane] = sum;
#pragma unroll
      for (int d = 0; d < 4; ++d) s_o[warp][d][lane] = acc[d];
      __syncthreads();
      if (warp < 4 && exists) {
        float top = -INFINITY, l = 0.f;
        float4 o = zero;
#pragma unroll
        for (int w = 0; w < TC_WARPS; ++w) top = fmaxf(top, s_m[w][lane]);
#pragma unroll
        for (int w = 0; w < TC_WARPS; ++w) {
          const float f = weight(s_m[w][lane], top);
          l += f * s_l[w][lane];
          add(o, f, s_o[w][warp][lane]);
        }
        store(row, (quad + warp) * 4, o, l);
      }
    }
    before += all;
  }
}

// How a call is launched: ranges, tiles of rows walked side by side.
struct TreePlan {
  int x, y, npt;
  bool whole;
  int64_t slot_bytes, bytes;
};
TreePlan plan_tree(const b2_ctx* ctx, int n_seqs, int max_q, int group, int nkv, int head_dim, int64_t max_len) {
  TreePlan p;
  p.npt = TR_ROWS / group;
  p.y = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((static_cast<int64_t>(max_q) + p.npt - 1) / p.npt, 8)));
  const int64_t most = std::max<int64_t>(1, static_cast<int64_t>(n_seqs) * nkv * ((max_len + TR_KEYS - 1) / TR_KEYS + TR_ITEM_UNITS) *
                                              ((static_cast<int64_t>(max_q) + p.npt * p.y - 1) / (p.npt * p.y)));
  p.x = static_cast<int>(std::min<int64_t>(most, std::max(1, ctx->num_sms * TR_CTAS_PER_SM / p.y)));
  // Contexts of at most TR_WHOLE_TILES tiles are not cut where there are CTAs for all of them.  (By the tables' width: the lengths are on the device.)
  p.whole = max_len <= TR_WHOLE_TILES * TR_KEYS && n_seqs > 0 && static_cast<int64_t>(n_seqs) * nkv * p.y <= ctx->num_sms * TR_CTAS_PER_SM;
  if (p.whole) p.x = n_seqs * nkv;
  p.slot_bytes = static_cast<int64_t>(head_dim == 128 ? Tree<128>::SLOT : Tree<64>::SLOT) * sizeof(float);
  p.bytes = p.whole ? 0 : static_cast<int64_t>(p.x) * p.y * (2 * p.slot_bytes + sizeof(int4));
  return p;
}

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    B2_CUDA(cudaFuncSetAttribute(tree_attention_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tree<128>::smem(TR_MAX_SEQS)));
    B2_CUDA(cudaFuncSetAttribute(tree_attention_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tree<64>::smem(TR_MAX_SEQS)));
    done[dev].store(true, std::memory_order_release);
  }
  return B2_OK;
}

}  // namespace

extern "C" {

int b2_tree_attention_supported(int nq, int nkv, int head_dim, int block_size) {
  return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= TR_ROWS && nkv <= 65535 && (head_dim == 64 || head_dim == 128) && block_size > 0 && block_size % 16 == 0;
}

int64_t b2_tree_attention_workspace(b2_ctx* ctx, int n_seqs, int max_q, int nq, int nkv, int head_dim, int block_size, int bt_width) {
  if (ctx == nullptr || n_seqs < 0 || n_seqs > TR_MAX_SEQS || max_q < 0 || bt_width < 0 || !b2_tree_attention_supported(nq, nkv, head_dim, block_size)) return -1;
  return plan_tree(ctx, n_seqs, max_q, nq / nkv, nkv, head_dim, static_cast<int64_t>(bt_width) * block_size).bytes;
}

int b2_tree_attention(b2_ctx* ctx, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int num_blocks, int block_size,
                      const int32_t* block_tables, int64_t bt_stride, int bt_width, const int32_t* cu_q, const int32_t* context_lens, const int64_t* tree_mask,
                      int64_t mask_stride, int mask_words, int n_seqs, int max_q, int tokens, int nq, int nkv, int head_dim, float scale, void* out,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n_seqs < 0 || tokens < 0 || nq <= 0 || nkv <= 0 || max_q < 0) return B2_ERR_ARG;
  if (tokens == 0) return B2_OK;
  if (!b2_tree_attention_supported(nq, nkv, head_dim, block_size)) return B2_ERR_UNSUPPORTED;
  if (!q || !k_cache || !v_cache || !cu_q || !out || (n_seqs > 0 && (!block_tables || !context_lens || !tree_mask))) return B2_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return B2_ERR_ARG;
  if (q_stride % 8 != 0 || q_stride < static_cast<int64_t>(nq) * head_dim || num_blocks <= 0 || bt_width <= 0 || bt_stride < bt_width || mask_words <= 0 ||
      mask_stride < mask_words)
    return B2_ERR_ARG;
  const int64_t max_len = static_cast<int64_t>(bt_width) * block_size;
  if (n_seqs > TR_MAX_SEQS) return b2::set_error(B2_ERR_SHAPE, "%d sequences, at most %d", n_seqs, TR_MAX_SEQS);
  const TreePlan p = plan_tree(ctx, n_seqs, max_q, nq / nkv, nkv, head_dim, max_len);
  // (tiles are counted in 32 bits: those of all sequences and heads, a pass for every gridDim.y tiles of rows)
  const int64_t passes = (static_cast<int64_t>(tokens) + p.npt * p.y - 1) / (p.npt * p.y) + n_seqs;
  if (static_cast<int64_t>(num_blocks) * block_size >= 1ll << 31 || max_len >= 1ll << 31 || passes * nkv * ((max_len + TR_KEYS - 1) / TR_KEYS + TR_ITEM_UNITS) >= 1ll << 31)
    return b2::set_error(B2_ERR_SHAPE, "%lld slots, tables of %lld tokens", static_cast<long long>(num_blocks) * block_size, static_cast<long long>(max_len));
  if (workspace_bytes < p.bytes || (p.bytes > 0 && workspace == nullptr)) return B2_ERR_ARG;
  const int rc = configure_once();
  if (rc != B2_OK) return rc;
  TreeArgs a{};
  a.v = static_cast<const uint16_t*>(v_cache);
  a.tables = block_tables;
  a.bt_stride = bt_stride;
  a.bt_width = bt_width;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.box = block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : 16;
  a.cu_q = cu_q;
  a.lens = context_lens;
  a.mask = tree_mask;
  a.mask_stride = mask_stride;
  a.words = mask_words;
  a.n_seqs = n_seqs;
  a.tokens = tokens;
  a.nq = nq;
  a.nkv = nkv;
  a.group = nq / nkv;
  a.npt = p.npt;
  a.negate = scale < 0.f ? b2::kUmmaNegateA : 0u;
  a.scale_log2 = b2::scale_size(scale);
  a.out = static_cast<uint16_t*>(out);
  a.whole = p.whole;
  a.parts = static_cast<float*>(workspace);
  a.joins = p.whole ? nullptr : reinterpret_cast<int4*>(static_cast<char*>(workspace) + 2 * p.x * p.y * p.slot_bytes);
  a.status = ctx->status_dev;
  CUtensorMap tmQ, tmK, tmV;
  const uint64_t width = static_cast<uint64_t>(nkv) * head_dim, slots = static_cast<uint64_t>(num_blocks) * block_size;
  int e = b2::encode_tmap_3d(&tmQ, q, head_dim, nq, tokens, q_stride, 64, a.group, a.npt);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmK, k_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e == B2_OK) e = b2::encode_tmap_2d(&tmV, v_cache, width, slots, static_cast<int64_t>(width), 64, a.box);
  if (e != B2_OK) return e;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  const size_t smem = head_dim == 128 ? Tree<128>::smem(n_seqs) : Tree<64>::smem(n_seqs);
  B2_CUDA(b2_launch(head_dim == 128 ? tree_attention_kernel<128> : tree_attention_kernel<64>, dim3(p.x, p.y), dim3(TR_THREADS), smem, on, tmQ, tmK, tmV, a));
  if (!p.whole)
    B2_CUDA(b2_launch(head_dim == 128 ? tree_combine_kernel<128> : tree_combine_kernel<64>, dim3(TC_CTAS_PER_SM * ctx->num_sms), dim3(TC_WARPS * 32), 0, on, a, p.x, p.y));
  return B2_OK;
}

}  // extern "C"
