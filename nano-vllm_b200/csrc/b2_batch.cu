// The inputs of a step of the model, built on the GPU from the requests' lengths: block tables, positions and slots.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// batch_inputs_kernel
//
// Row i has c = cached[i] tokens in the cache and is to have w = wanted[i].  With have = ceil(c / block_size), want = ceil(w / block_size):
//   add  = max(0, w - c)        tokens of this step        need = max(0, want - have)  blocks from the free stack
//                                                          back = max(0, have - want)  blocks onto it
// The stack's top is what the rows give back, in their order, and below it what was free; the granted rows take from the top, in
// their order.  Every block, slot and position follows from the prefix sums of add, need and back, so that each CTA forms these
// sums for the whole batch (a few KB from L2) and then does its share of the tokens, of the new table entries and of the stack: one
// launch without any exchange between CTAs.  Nothing that one CTA reads is written by another: taken blocks go to table entries
// past `have`, given ones are read from entries past `want` of rows that take none, and the stack is written above num_free.
//
// Bound: latency in steps of up to 16384 tokens (device time one after the other: one row 3.4 us, 512 rows that grow or finish 6.6, 16384 tokens 4.5).  Beyond, the
// places written, 12 bytes each, those behind the last token too: room for 2^20 takes 12 us, for 2^24 62 us (3.2 TB/s, what 64 CTAs store).
// ---------------------------------------------------------------------------
constexpr int BI_THREADS = 512;
constexpr int BI_MAX_ROWS = 8192;
constexpr int BI_ARRAYS = 5;  // shared memory: cached, wanted, and the prefix sums of tokens, of blocks taken and given back
constexpr size_t batch_smem(int n) { return static_cast<size_t>(BI_ARRAYS) * (n + 1) * sizeof(int); }

struct BatchArgs {
  int32_t* tables;
  int64_t bt_stride;
  int bt_width;
  const int32_t *cached, *wanted;
  int n;
  int32_t* free_blocks;
  int capacity;
  const int32_t* num_free;
  int block_size;
  int64_t num_slots;
  int max_tokens;
  const int64_t* mask;
  int64_t mask_stride;
  int words;
  int64_t* positions;
  int32_t *slots, *cu_q, *cu_k, *last, *lens, *num_free_out;
};

struct Sums {
  int x, y, z;
};

// exclusive prefix sums over the block's threads; total: over all of them
__device__ __forceinline__ Sums scan(Sums v, Sums& total, int (*s_warp)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, in.x, o), y = __shfl_up_sync(0xffffffffu, in.y, o), z = __shfl_up_sync(0xffffffffu, in.z, o);
    if (lane >= o) in = {in.x + x, in.y + y, in.z + z};
  }
  __syncthreads();  // (the sums of the scan before have been read)
  if (lane == 31) {
    s_warp[warp][0] = in.x;
    s_warp[warp][1] = in.y;
    s_warp[warp][2] = in.z;
  }
  __syncthreads();
  Sums before = {0, 0, 0};
  total = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < BI_THREADS / 32; ++w) {
    if (w == warp) before = total;
    total = {total.x + s_warp[w][0], total.y + s_warp[w][1], total.z + s_warp[w][2]};
  }
  return {before.x + in.x - v.x, before.y + in.y - v.y, before.z + in.z - v.z};
}

// the row whose range [sums[row], sums[row + 1]) holds i, for sums[0] <= i < sums[n]
__device__ __forceinline__ int row_of(const int* sums, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(BI_THREADS) batch_inputs_kernel(const BatchArgs a) {
  extern __shared__ int s_rows[];
  int *const s_c = s_rows, *const s_w = s_c + a.n + 1, *const s_tok = s_w + a.n + 1, *const s_need = s_tok + a.n + 1, *const s_back = s_need + a.n + 1;
  __shared__ int s_warp[BI_THREADS / 32][3];
  const int tid = threadIdx.x;
  b2::pdl_wait();

  const int bs = a.block_size, full = a.bt_width * bs;  // (the host has checked that n * full is below 2^31)
  auto blocks = [&](int tokens) { return static_cast<int>((static_cast<uint32_t>(tokens) + bs - 1) / bs); };  // (the sum may pass 2^31, not 2^32)
  const int per = (a.n + BI_THREADS - 1) / BI_THREADS, r0 = min(a.n, tid * per), r1 = min(a.n, r0 + per);
  Sums mine = {0, 0, 0};
  for (int r = r0; r < r1; ++r) {
    int c = __ldg(a.cached + r), w = __ldg(a.wanted + r);
    if (c < 0 || c > full || w < 0 || w > full) c = w = 0;  // lengths that no row of the table can hold: a row without tokens
    s_c[r] = c;
    s_w[r] = w;
    const int d = blocks(w) - blocks(c);
    mine = {mine.x + max(0, w - c), mine.y + max(0, d), mine.z + max(0, -d)};
  }
  Sums total, at = scan(mine, total, s_warp);
  const int num_free = max(0, min(__ldg(a.num_free), a.capacity)), top = num_free + total.z;

  // which rows are served: tokens and blocks are asked for in the order of the rows
  int taken = 0, len_sum = 0;
  {
    Sums run = at;
    int counted = 0, need_sum = 0;
    for (int r = r0; r < r1; ++r) {
      const int c = s_c[r], w = s_w[r], d = blocks(w) - blocks(c), add = max(0, w - c), need = max(0, d);
      run.x += add;
      run.y += need;
      const bool fits = run.x <= a.max_tokens, granted = fits && (need == 0 || run.y <= top);
      counted += fits ? add : 0;
      need_sum += granted ? need : 0;
      len_sum += w < c || granted ? w : c;
    }
    Sums all, first = scan({counted, need_sum, len_sum}, all, s_warp);
    run = at;
    for (int r = r0; r < r1; ++r) {
      const int c = s_c[r], w = s_w[r], d = blocks(w) - blocks(c), add = max(0, w - c), need = max(0, d);
      s_tok[r] = first.x;
      s_need[r] = first.y;
      s_back[r] = run.z;
      if (blockIdx.x == 0) {
        a.cu_q[r] = first.x;
        a.cu_k[r] = first.z;
      }
      run = {run.x + add, run.y + need, run.z + max(0, -d)};
      const bool fits = run.x <= a.max_tokens, granted = fits && (need == 0 || run.y <= top);
      const int len = w < c || granted ? w : c;
      if (!granted && add > 0) s_w[r] = -1;  // its tokens get no slots
      first = {first.x + (fits ? add : 0), first.y + (granted ? need : 0), first.z + len};
      if (blockIdx.x == 0) {
        a.lens[r] = len;
        a.last[r] = max(0, first.x - 1);
      }
    }
    taken = all.y;
    if (tid == 0) {
      s_tok[a.n] = all.x;
      s_need[a.n] = all.y;
      s_back[a.n] = total.z;
      if (blockIdx.x == 0) {
        a.cu_q[a.n] = all.x;
        a.cu_k[a.n] = all.z;
        *a.num_free_out = min(a.capacity, top - taken);
      }
    }
  }
  __syncthreads();

  // place k of what the rows give back, and place i of the stack with that on top
  auto returned = [&](int k) {
    const int r = row_of(s_back, a.n, k);
    return a.tables[static_cast<int64_t>(r) * a.bt_stride + blocks(s_w[r]) + k - s_back[r]];
  };
  auto stacked = [&](int i) { return i < num_free ? a.free_blocks[i] : returned(i - num_free); };
  const int first = blockIdx.x * BI_THREADS + tid, step = gridDim.x * BI_THREADS;
  for (int t = first; t < a.max_tokens; t += step) {
    int64_t position = 0;
    int slot = -1;
    if (t < s_tok[a.n]) {
      const int r = row_of(s_tok, a.n, t), c = s_c[r], i = t - s_tok[r], place = c + i, j = place / bs;
      position = place;
      if (a.mask != nullptr) {
        int sees = 0;  // of the row's own nodes
        for (int w = 0, left = s_tok[r + 1] - s_tok[r]; w < a.words && left > 0; ++w, left -= 64)
          sees += __popcll(__ldg(reinterpret_cast<const unsigned long long*>(a.mask + t * a.mask_stride + w)) & (left < 64 ? (1ull << left) - 1 : ~0ull));
        position = c + max(0, sees - 1);
      }
      if (s_w[r] >= 0) {
        const int have = blocks(c);
        const int block = j < have ? a.tables[static_cast<int64_t>(r) * a.bt_stride + j] : stacked(top - 1 - s_need[r] - (j - have));
        const int64_t s = static_cast<int64_t>(block) * bs + (place - j * bs);
        if (block >= 0 && s < a.num_slots) slot = static_cast<int>(s);
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  for (int k = first; k < taken; k += step) {
    const int r = row_of(s_need, a.n, k);
    a.tables[static_cast<int64_t>(r) * a.bt_stride + blocks(s_c[r]) + k - s_need[r]] = stacked(top - 1 - k);
  }
  for (int i = num_free + first; i < min(a.capacity, top - taken); i += step) a.free_blocks[i] = returned(i - num_free);
  b2::pdl_release_results();  // later kernels may read the lengths and tables ahead of their dependency wait
}

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    B2_CUDA(cudaFuncSetAttribute(batch_inputs_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, batch_smem(BI_MAX_ROWS)));
    done[dev].store(true, std::memory_order_release);
  }
  return B2_OK;
}

}  // namespace

extern "C" int b2_batch_inputs(int32_t* block_tables, int64_t bt_stride, int bt_width, const int32_t* cached_lens, const int32_t* seq_lens, int n,
                               int32_t* free_blocks, int free_capacity, const int32_t* num_free, int block_size, int64_t num_slots, int max_tokens,
                               const int64_t* tree_mask, int64_t mask_stride, int mask_words, int64_t* positions, int32_t* slot_mapping, int32_t* cu_seqlens_q,
                               int32_t* cu_seqlens_k, int32_t* last_token_index, int32_t* context_lens, int32_t* num_free_out, void* stream) {
  if (n < 0 || free_capacity < 0 || block_size <= 0 || num_slots <= 0 || max_tokens < 0 || bt_width < 0) return B2_ERR_ARG;
  if (n > 0 && (bt_width <= 0 || bt_stride < bt_width || !block_tables || !cached_lens || !seq_lens || !last_token_index || !context_lens)) return B2_ERR_ARG;
  if (!num_free || !num_free_out || !cu_seqlens_q || !cu_seqlens_k || (free_capacity > 0 && !free_blocks)) return B2_ERR_ARG;
  if (max_tokens > 0 && (!positions || !slot_mapping)) return B2_ERR_ARG;
  if (tree_mask != nullptr && (mask_words <= 0 || mask_stride < mask_words)) return B2_ERR_ARG;
  if (n > BI_MAX_ROWS) return b2::set_error(B2_ERR_SHAPE, "%d rows, at most %d", n, BI_MAX_ROWS);
  constexpr int64_t limit = (1ll << 31) - 1;
  if (static_cast<int64_t>(n) * bt_width > limit / block_size || static_cast<int64_t>(n) * bt_width + free_capacity > limit || num_slots > limit || max_tokens > 1 << 30)
    return b2::set_error(B2_ERR_SHAPE, "lengths, blocks, slots and tokens must each add up to less than 2^31");
  const int rc = configure_once();
  if (rc != B2_OK) return rc;
  const BatchArgs a{block_tables, bt_stride, bt_width, cached_lens, seq_lens, n, free_blocks, free_capacity, num_free, block_size, num_slots, max_tokens,
                    tree_mask, mask_stride, mask_words, positions, slot_mapping, cu_seqlens_q, cu_seqlens_k, last_token_index, context_lens, num_free_out};
  // a thread for each token, and for every fourth block that the tables have room for: how many of them move is known on the device only (512 rows of 257
  // blocks, a tenth of which finish and give 6500 back: 10.6 us with a CTA for every 512 tokens, 6.3 so)
  const int64_t work = std::max<int64_t>(max_tokens, static_cast<int64_t>(n) * bt_width / 4);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(64, (work + BI_THREADS - 1) / BI_THREADS)));
  B2_CUDA(b2_launch(batch_inputs_kernel, dim3(grid), dim3(BI_THREADS), batch_smem(n), static_cast<cudaStream_t>(stream), a));
  return B2_OK;
}
