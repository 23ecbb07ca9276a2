// A step of beam search: the best continuations of each request, and what its beams have in the cache following them.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// beam_scan_kernel, beam_pick_kernel
//
// A continuation of beam b by token v has the score s_b + x_bv - log sum_u exp x_bu.  Within a beam the order is that of the logits, so that
// one pass over them gives all that is needed: the running maximum and sum of each row, and its K best tokens.
//
// beam_scan_kernel: the rows in tiles of 16 KB, dealt in contiguous equal ranges to the CTAs, so that every SM streams whatever the
// batch.  A thread keeps its own maximum and sum.  Candidates go to a list in shared memory: of the first tile of a range those that reach
// the K-th best of the threads' maxima (a lower bound of the K-th best logit), later those above the bound, which rises when the list is cut back
// to K.  A key is (logit, lowest token first), so that keys are never equal and the list is bounded: a bound that c threads' maxima reach is
// reached by at most 32 c logits.
//
// beam_pick_kernel: a CTA per request joins its rows' parts.  Scores are formed in 64 bits.  The sums' error (exponentials of the hardware, sums
// in 32 bits) could turn the order of continuations of two beams that lie closer than BS_NEAR; where that is so among the K + 1 best, those
// beams' sums are formed again in 64 bits from the logits.
//
// Bound: HBM, every logit read once.
// ---------------------------------------------------------------------------
constexpr int BS_THREADS = 256, BS_VECTORS = 4, BS_CTAS_PER_SM = 4, BS_GROUP = 4;
constexpr int BS_TILE_BYTES = BS_THREADS * BS_VECTORS * 16;
constexpr int BS_MAX_PICKS = 64, BS_MAX_BEAMS = 32;
constexpr int BP_THREADS = 512, BP_LISTS = 256;
constexpr int BS_COLLECT = 1536, BP_RANKED = 192;  // candidates that a request collects, and that it ranks without another bound
constexpr double BS_NEAR = 4e-6;

struct ScanArgs {
  const void* logits;
  int64_t ld;
  int rows, beams, vocab, picks;
  int tiles, parts;  // per row: tiles, most parts
  int capacity;      // of the list of candidates
  const float* scores;
  const uint8_t* finished;
  uint64_t* keys;  // [rows][parts][picks], best first, 0: none
  double2* sums;   // [rows][parts] (M, sum of 2^(x log2(e) - M)); M is a whole number, -inf where there is nothing
};

__device__ __forceinline__ uint32_t ordered(float x) {  // unsigned order = order of the numbers; -0 is 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(float x, int token) { return (static_cast<uint64_t>(ordered(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(token)); }
__device__ __forceinline__ int token_of(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LOG2E_64 = 1.4426950408889634, LN2_64 = 0.6931471805599453;
constexpr float BS_PLAIN = 65536.f;  // below this size x log2(e) is formed in 32 bits
// 2^x of a whole number x <= 0, exactly; 0 below the normal range (and for NaN, the difference of two -inf)
__device__ __forceinline__ double power_of_two(double x) { return x > -1023.0 ? __longlong_as_double(static_cast<long long>(1023 + static_cast<int>(x)) << 52) : 0.0; }

// NaN counts as -inf, +inf as the largest number
__device__ __forceinline__ float plain_number(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float most() { return FLT_MAX; }
  static __device__ __forceinline__ float one(const float* p) { return plain_number(__ldg(p)); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
template <>
struct Logits<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float most() { return b2::bf16_hi(0x7f7f0000u); }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return fminf(fmaxf(__bfloat162float(*p), -INFINITY), most()); }
  static __device__ __forceinline__ uint32_t max2(uint32_t x, uint32_t y) {
    const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) { b2::unpack8(v, f); }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const uint32_t w = max2(max2(v.x, v.y), max2(v.z, v.w));
    return fmaxf(b2::bf16_lo(w), b2::bf16_hi(w));
  }
};

// The 16 bytes at `chunk` (counted from the 16-byte boundary at or before the row), -inf in the places that are not the row's.
template <typename T>
__device__ __noinline__ uint4 load_chunk(const T* row, int vocab, int64_t first) {  // first: the row's element at which the chunk begins, may be < 0
  constexpr int N = Logits<T>::N;
  if (first >= 0 && first + N <= vocab) return __ldg(reinterpret_cast<const uint4*>(row + first));
  uint32_t w[4] = {0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
  if constexpr (N == 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = 0xff80ff80u;
  }
  if (first < vocab && first + N > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int64_t i = first + e;
      if (i < 0 || i >= vocab) continue;
      if constexpr (N == 8) {
        const uint32_t x = __ldg(reinterpret_cast<const unsigned short*>(row) + i);
        w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | (x << 16) : (w[e >> 1] & 0xffff0000u) | x;
      } else {
        w[e] = __float_as_uint(__ldg(reinterpret_cast<const float*>(row) + i));
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The list of candidates of a CTA
struct List {
  uint64_t *keys, *best;  // [capacity], [BS_MAX_PICKS]
  int* count;             // of those that were to go in: may be past the capacity
  int capacity;
  __device__ __forceinline__ void push(uint64_t key) const {
    const int at = atomicAdd(count, 1);
    if (at < capacity) keys[at] = key;
  }
  // All threads: the k best of the n keys stay, in order.  Every thread counts the keys before its own.  Returns how many there are.
  __device__ __noinline__ int rank(int n, int k) const {
    for (int i = threadIdx.x; i < n; i += BS_THREADS) {
      const uint64_t mine = keys[i];
      int before = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) before += keys[j] > mine ? 1 : 0;
      if (before < k) best[before] = mine;
    }
    __syncthreads();
    const int left = min(n, k);
    if (static_cast<int>(threadIdx.x) < left) keys[threadIdx.x] = best[threadIdx.x];
    if (threadIdx.x == 0) *count = left;
    __syncthreads();
    return left;
  }
  // All threads: those of the n keys stay, in no order, whose logits reach the bound.
  __device__ __noinline__ int filter(int n, float bound) const {
    const uint64_t least = static_cast<uint64_t>(ordered(bound)) << 32;
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    // in steps of the block: what a step writes lies before what later ones read
    for (int i0 = 0; i0 < n; i0 += BS_THREADS) {
      const uint64_t mine = i0 + static_cast<int>(threadIdx.x) < n ? keys[i0 + threadIdx.x] : 0;
      __syncthreads();
      if (mine >= least && mine != 0) keys[atomicAdd(count, 1)] = mine;
      __syncthreads();
    }
    const int left = *count;
    __syncthreads();
    return left;
  }
};

// (Out of line: rare, or little beside the loop over the tiles, which has to fit the instruction cache.)
// All threads: the candidates among tokens first .. last, for which there was no room (many equal logits, or a row that rises all along): 256 at a time.
template <typename T>
__device__ __noinline__ int overflow(const List list, const T* p, int vocab, int k, int count, int first, int last) {
  if (threadIdx.x == 0) *list.count = count;
  __syncthreads();
  if (count >= k) count = list.rank(count, k);
  for (; first < last; first += BS_THREADS) {
    const int token = first + threadIdx.x;
    const uint64_t least = count >= k ? list.keys[k - 1] : 0;
    __syncthreads();
    if (token >= 0 && token < vocab) {
      const float f = Logits<T>::one(p + token);
      if (f > -INFINITY && key_of(f, token) > least) list.push(key_of(f, token));
    }
    __syncthreads();
    count = list.rank(*list.count, k);
  }
  return count;
}
// largest logit of a thread's part of a tile
template <typename T>
__device__ __noinline__ float tile_maximum(const T* p, int vocab, int token0) {
  constexpr int N = Logits<T>::N;
  float top = -INFINITY;
  for (int i = 0; i < BS_VECTORS * N; ++i) {
    const int token = token0 + i / N * (BS_THREADS * N) + i % N;
    if (token >= 0 && token < vocab) top = fmaxf(top, Logits<T>::one(p + token));
  }
  return top;
}
// sum of 2^(x log2(e) - ref) over it, in 64 bits
template <typename T>
__device__ __noinline__ double exact_sum(const T* p, int vocab, int token0, double ref) {
  constexpr int N = Logits<T>::N;
  double sum = 0.0;
  for (int i = 0; i < BS_VECTORS * N; ++i) {
    const int token = token0 + i / N * (BS_THREADS * N) + i % N;
    if (token >= 0 && token < vocab) sum += exp2(__dmul_rn(Logits<T>::one(p + token), LOG2E_64) - ref);
  }
  return sum;
}
// All threads: a number that the numbers of at least k of them reach, quickly: each warp's ceil(k / warps)-th largest, and the least of those.
__device__ __noinline__ float reached_by(float x, int k, float* of_warps) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (k + BS_THREADS / 32 - 1) / (BS_THREADS / 32);
  for (int i = 1; i < each; ++i) {  // the largest is taken out
    const unsigned best = __reduce_max_sync(0xffffffffu, ordered(x));
    const unsigned who = __ballot_sync(0xffffffffu, ordered(x) == best);
    if (lane == __ffs(who) - 1) x = -INFINITY;
  }
  const unsigned best = __reduce_max_sync(0xffffffffu, ordered(x));
  if (lane == 0) of_warps[warp] = number_of(best);
  __syncthreads();
  x = of_warps[0];
#pragma unroll
  for (int w = 1; w < BS_THREADS / 32; ++w) x = fminf(x, of_warps[w]);
  __syncthreads();
  return x;
}
// All threads: the k-th largest of one number each.  The warps sort theirs, and every thread finds its own's place in the others.
__device__ __noinline__ float kth_of_threads(float x, int k, float* sorted, float* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int j = n >> 1; j > 0; j >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, j);
      x = ((lane & j) == 0) == ((lane & n) == 0) ? fmaxf(x, y) : fminf(x, y);
    }
  sorted[tid] = x;
  __syncthreads();
  int rank = lane;
  for (int w = 0; w < BS_THREADS / 32; ++w) {
    if (w == warp) continue;
    int lo = 0;  // how many of warp w come before
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
      const float y = sorted[w * 32 + lo + step - 1];
      if (y > x || (y == x && w < warp)) lo += step;
    }
    const float y = sorted[w * 32 + lo];
    if (y > x || (y == x && w < warp)) ++lo;
    rank += lo;
  }
  if (rank == k - 1) *found = x;
  __syncthreads();
  return *found;
}

// Ranges of `total` tiles: CTA x of X
struct ScanDeal {
  int base, rem;
  __device__ __forceinline__ ScanDeal(int total, int X) : base(total / X), rem(total % X) {}
  __device__ __forceinline__ int begin_of(int x) const { return x * base + min(x, rem); }
  __device__ __forceinline__ int cta_of(int t) const {
    const int big = rem * (base + 1);
    return t < big ? t / (base + 1) : rem + (t - big) / base;
  }
};

template <typename T>
__global__ void __launch_bounds__(BS_THREADS, BS_CTAS_PER_SM) beam_scan_kernel(const ScanArgs a) {
  constexpr int N = Logits<T>::N, TILE = BS_THREADS * BS_VECTORS * N;
  extern __shared__ __align__(16) uint64_t s_keys[];
  __shared__ uint64_t s_best[BS_MAX_PICKS];
  __shared__ int s_count;
  __shared__ float s_top[BS_THREADS], s_bound;
  __shared__ double s_ref[BS_THREADS / 32], s_sum[BS_THREADS / 32];
  List list{s_keys, s_best, &s_count, a.capacity};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.picks;
  const ScanDeal deal(a.rows * a.tiles, gridDim.x);
  int u = deal.begin_of(blockIdx.x);
  const int end = deal.begin_of(blockIdx.x + 1);
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  while (u < end) {
    const int row = u / a.tiles, t0 = u - row * a.tiles, t1 = min(a.tiles, t0 + end - u);
    u += t1 - t0;
    if (!(a.scores[row] > -INFINITY) || (a.finished != nullptr && a.finished[row] != 0)) continue;  // (it has one continuation or none)
    const int part = blockIdx.x - deal.cta_of(row * a.tiles);  // the CTA that holds the row's first tile is the first of its parts
    const T* p = static_cast<const T*>(a.logits) + row * a.ld;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));  // tiles begin at the 16-byte boundary before the row
    const int limit = max(K + 32, min(2 * K + 64, a.capacity / 2));  // candidates at which the list is cut
    auto load = [&](int tile, uint4 (&v)[BS_VECTORS]) {
      const int64_t first = static_cast<int64_t>(tile) * TILE - shift;
      if (first >= 0 && first + TILE <= a.vocab) {
        const uint4* q = reinterpret_cast<const uint4*>(p + first) + tid;
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) v[i] = __ldg(q + i * BS_THREADS);
      } else {
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) v[i] = load_chunk(p, a.vocab, first + (i * BS_THREADS + tid) * N);
      }
    };
    uint4 next[BS_VECTORS];
    load(t0, next);
    float bound = INFINITY;     // logits from here on are candidates; not known before the first tile has been read
    float highest = -INFINITY;  // of the thread's logits
    // The sum's reference is a power of two, so that raising it is exact, and x log2(e) - M is one rounding of an exact product.
    double ref = -INFINITY, sum = 0.0;
    float ref_low = -INFINITY;  // ref as far as 32 bits go
    auto raise = [&](double to) {
      if (to > ref) {
        sum *= power_of_two(ref - to);
        ref = to;
        ref_low = static_cast<float>(to);
      }
    };
    if (tid == 0) s_count = 0;
    int count = 0;
    // The first tile, and then BS_GROUP at a time: what they hold is noted by vectors, and looked at when they are through.
#pragma unroll 1
    for (int tile = t0; tile < t1;) {
      const int group = tile, last = tile == t0 ? t0 + 1 : min(t1, tile + BS_GROUP);
      unsigned reach = 0, odd = 0;  // vectors whose largest reaches the bound; tiles with infinities, NaN or very large numbers
      float best[BS_VECTORS];
#pragma unroll 1
      for (; tile < last; ++tile) {
        uint4 now[BS_VECTORS];
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) now[i] = next[i];
        if (tile + 1 < t1) load(tile + 1, next);
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) best[i] = Logits<T>::largest(now[i]);
        const float top = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
        const float mine = rintf(top * LOG2E);
        if (mine > ref_low && top < BS_PLAIN) raise(mine);
        uint64_t sums[2] = {};
        const uint64_t minus = b2::pair_of(-ref_low, -ref_low), scale = b2::pair_of(LOG2E, LOG2E);
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) {
          float f[N];
          Logits<T>::unpack(now[i], f);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            float x, y;
            b2::fma_pair(x, y, b2::pair_of(f[e], f[e + 1]), scale, minus);
            sums[(e >> 1) & 1] = b2::add_pair(sums[(e >> 1) & 1], b2::pair_of(b2::ex2(x), b2::ex2(y)));
          }
          if (best[i] >= bound) reach |= 1u << ((tile - group) * BS_VECTORS + i);
        }
        float x, y;
        b2::halves_of(b2::add_pair(sums[0], sums[1]), x, y);
        // (NaN among the logits makes the sum one; with nothing but -inf so far it is one as well, or has nothing to add)
        if (fabsf(top) < BS_PLAIN && x + y < INFINITY) sum += x + y;
        else if (top != -INFINITY) odd |= 1u << (tile - group);
        highest = fmaxf(highest, top < INFINITY ? top : -INFINITY);
      }
      // ---- once a group ----
      for (; odd != 0; odd &= odd - 1) {
        const int t = __ffs(odd) - 1, token0 = (group + t) * TILE - shift + tid * N;
        const float top = tile_maximum<T>(p, a.vocab, token0);
        if (top > -INFINITY) {
          raise(rint(__dmul_rn(top, LOG2E_64)));
          sum += exact_sum<T>(p, a.vocab, token0, ref);
        }
        highest = fmaxf(highest, top);
      }
      if (group == t0) {
        bound = reached_by(highest, K, s_top);
        if (bound == -INFINITY) bound = fmaxf(-FLT_MAX, kth_of_threads(highest, K, s_top, &s_bound));
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i)
          if (best[i] >= bound) reach |= 1u << i;
      }
      for (; reach != 0; reach &= reach - 1) {
        const int v = __ffs(reach) - 1, token = (group + v / BS_VECTORS) * TILE - shift + (v % BS_VECTORS * BS_THREADS + tid) * N;
        const uint4 w = load_chunk(p, a.vocab, token);  // (from L2, where it has just been)
        float f[N];
        Logits<T>::unpack(w, f);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (f[e] >= bound) list.push(key_of(fminf(f[e], Logits<T>::most()), token + e));
      }
      __syncthreads();
      const int seen = s_count, fresh = seen - count;
      __syncthreads();  // (the next group's may go in)
      if (seen <= a.capacity) {
        count = seen;
      } else {
        count = overflow<T>(list, p, a.vocab, K, count, group * TILE - shift, last * TILE - shift);
        if (count >= K) bound = fmaxf(bound, number_of(static_cast<uint32_t>(s_keys[K - 1] >> 32) + 1));
      }
      if (tile < t1 && fresh > K / 2) {
        // Later tokens have to be above what K threads have seen: as high, they would come behind those.
        const float higher = group == t0 && bound > -FLT_MAX ? bound : reached_by(highest, K, s_top);
        if (higher >= bound) {
          if (count > limit) count = list.filter(count, higher);
          bound = number_of(ordered(higher) + 1);
        }
      }
    }
    // ---- the part: maximum and sum, and the K best in order ----
    if (count > 2 * K + 32) {
      const float higher = kth_of_threads(highest, K, s_top, &s_bound);
      if (higher >= bound) count = list.filter(count, higher);
    }
    count = list.rank(count, K);
    const int64_t at = static_cast<int64_t>(row) * a.parts + part;
    if (tid < K) a.keys[at * K + tid] = tid < count ? s_keys[tid] : 0;
    double top = ref;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_ref[warp] = top;
    __syncthreads();
    top = s_ref[0];
#pragma unroll
    for (int w = 1; w < BS_THREADS / 32; ++w) top = fmax(top, s_ref[w]);
    double all = sum * power_of_two(ref - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) s_sum[warp] = all;
    __syncthreads();
    if (tid == 0) {
      all = 0.0;
      for (int w = 0; w < BS_THREADS / 32; ++w) all += s_sum[w];
      a.sums[at] = make_double2(top, all);
    }
  }
}

struct PickArgs {
  ScanArgs scan;
  int grid;  // of the scan
  int eos;   // -1: none
  float* scores;
  int32_t* parents;
  int64_t* tokens;
  uint8_t* finished;
};
struct Candidate {
  double score;
  float x;
  int beam, token;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return a.score > b.score || (a.score == b.score && (a.beam < b.beam || (a.beam == b.beam && a.token < b.token)));
}

template <typename T>
__global__ void __launch_bounds__(BP_THREADS) beam_pick_kernel(const PickArgs a) {
  const ScanArgs& s = a.scan;
  constexpr int WARPS = BP_THREADS / 32;
  __shared__ double s_total[BS_MAX_BEAMS], s_score[BS_MAX_BEAMS], s_sum[WARPS], s_ref[BS_MAX_BEAMS];
  __shared__ int s_parts[BS_MAX_BEAMS + 1], s_kind[BS_MAX_BEAMS], s_again[BS_MAX_BEAMS], s_tally[32], s_count, s_any, s_reach, s_list[BP_LISTS];
  __shared__ uint32_t s_low, s_high;
  __shared__ Candidate s_got[BS_COLLECT], s_best[BS_MAX_PICKS + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = s.beams, K = s.picks, row0 = blockIdx.x * B;
  const ScanDeal deal(s.rows * s.tiles, a.grid);
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  if (warp == 0) {
    int parts = 0;
    if (lane < B) {
      const float score = s.scores[row0 + lane];
      const bool there = score > -INFINITY, ended = s.finished != nullptr && s.finished[row0 + lane] != 0;
      s_score[lane] = score;
      s_kind[lane] = !there ? 0 : ended ? 1 : 2;
      s_again[lane] = 0;
      const int first = (row0 + lane) * s.tiles;
      parts = !there ? 0 : ended ? 1 : deal.cta_of(first + s.tiles - 1) - deal.cta_of(first) + 1;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, parts, o);
      if (lane >= o) parts += up;
    }
    if (lane < B) s_parts[lane + 1] = parts;
    if (lane == 0) {
      s_parts[0] = s_count = s_any = s_reach = 0;
      s_low = 0xffffffffu;
      s_high = 0;
    }
  }
  if (tid < 32) s_tally[tid] = 0;
  __syncthreads();
  const int lists = s_parts[B];
  auto beam_of = [&](int list) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_parts[mid] <= list) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  // entry `depth` of a list of beam b: its key, 0 where there is none
  auto key_at = [&](int b, int list, int depth) -> uint64_t {
    if (s_kind[b] == 1) return depth == 0 ? 1 : 0;
    return depth < K ? s.keys[(static_cast<int64_t>(row0 + b) * s.parts + list - s_parts[b]) * K + depth] : 0;
  };
  auto candidate = [&](int b, uint64_t key) {
    if (s_kind[b] == 1) return Candidate{s_score[b], 0.f, b, -1};
    const float x = number_of(static_cast<uint32_t>(key >> 32));
    return Candidate{s_score[b] + (static_cast<double>(x) - s_total[b]), x, b, token_of(key)};
  };
  // ---- the lists' first entries, while the rows' sums are on their way ----
  constexpr int MOST = 8;  // entries of a thread
  const bool all_here = lists * K <= MOST * BP_THREADS;
  const int deep = lists > 0 ? (all_here ? K : (K + lists) / lists) : 0, n = lists * deep;
  uint64_t head[MOST];
  int of[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int g = tid + i * BP_THREADS;
    head[i] = 0;
    of[i] = 0;
    if (g < n) {
      const int list = all_here ? g / K : g % lists;
      of[i] = beam_of(list);
      head[i] = key_at(of[i], list, all_here ? g - list * K : g / lists);
    }
  }
  for (int b = warp; b < B; b += WARPS) {
    if (s_kind[b] != 2) continue;
    const int parts = s_parts[b + 1] - s_parts[b];
    const double2* sums = s.sums + static_cast<int64_t>(row0 + b) * s.parts;
    double top = -INFINITY, all = 0.0;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const double2 mine = i0 + lane < parts ? sums[i0 + lane] : make_double2(-INFINITY, 0.0);
      double higher = fmax(top, mine.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) higher = fmax(higher, __shfl_xor_sync(0xffffffffu, higher, o));
      all = all * power_of_two(top - higher) + mine.y * power_of_two(mine.x - higher);
      top = higher;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) {
      s_ref[b] = top;
      // log2(e) has 24 bits in the sum's exponents, which makes them this much too large; what carries the sum lies near M
      const double off = fabs(top) < 2 * BS_PLAIN ? top * (static_cast<double>(LOG2E) * LN2_64 - 1.0) : 0.0;
      s_total[b] = (top - off) * LN2_64 + log(all);
    }
  }
  __syncthreads();
  // All threads: a number that `enough` of the entries reach, and not many more than `most`; 0 where there are not as many.  Entries are 0 where there are none.
  auto reached = [&](const uint32_t (&mine)[MOST], int enough, int most) {
    uint32_t low = 0xffffffffu, high = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (mine[i] != 0) {
        low = min(low, mine[i]);
        high = max(high, mine[i]);
      }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0 && high != 0) {
      atomicMin(&s_low, low);
      atomicMax(&s_high, high);
    }
    __syncthreads();
    low = s_low;
    high = s_high;
    if (high == 0) return 0u;
    // the bits that all of them have in common are the bound's
    const int bits = low == high ? 0 : 32 - __clz(low ^ high);
    uint32_t reach = bits == 32 ? 0u : low >> bits << bits;
    bool any = false;
    for (int bit = bits - 1; bit >= 0; --bit) {
      const uint32_t c = reach | (1u << bit);
      int count = 0;
#pragma unroll
      for (int i = 0; i < MOST; ++i) count += __popc(__ballot_sync(0xffffffffu, mine[i] >= c));
      if (lane == 0 && count > 0) atomicAdd(s_tally + bit, count);
      __syncthreads();
      const int all = s_tally[bit];
      if (all < enough) continue;
      reach = c;
      any = true;
      if (all <= most) break;
    }
    return any ? reach : 0u;
  };
  // ---- a bound that at least K + 1 of the entries reach ----
  uint32_t t = 0;
  {
    uint32_t mine[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) mine[i] = head[i] != 0 ? ordered(static_cast<float>(candidate(of[i], head[i]).score)) : 0u;
    t = reached(mine, K + 1, K + 16);
  }
  // (a little lower: what lies as near as the sums' error belongs to it)
  auto below = [&](uint32_t reach) {
    if (reach <= 0x00800000u) return static_cast<double>(-INFINITY);
    const double x = number_of(reach);
    return x - 2 * BS_NEAR - 2.4e-7 * fabs(x);
  };
  double least = below(t);
  // ---- the entries that reach it ----
  if (all_here) {
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      if (head[i] == 0) continue;
      const Candidate c = candidate(of[i], head[i]);
      if (c.score >= least) {
        const int at = atomicAdd(&s_count, 1);
        if (at < BS_COLLECT) s_got[at] = c;
      }
    }
  } else {
    // of the lists whose first entry does; a warp takes a list, 32 entries at a time
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (tid + i * BP_THREADS < lists && head[i] != 0 && candidate(of[i], head[i]).score >= least) {
        const int at = atomicAdd(&s_reach, 1);
        if (at < BP_LISTS) s_list[at] = tid + i * BP_THREADS;
      }
    __syncthreads();
    const int reach = s_reach;
    if (reach <= BP_LISTS) {
      for (int l = warp; l < reach; l += WARPS) {
        const int list = s_list[l], b = beam_of(list);
        for (int d = 0; d < K; d += 32) {
          const uint64_t key = key_at(b, list, d + lane);
          Candidate c{};
          bool reaches = key != 0;
          if (reaches) {
            c = candidate(b, key);
            reaches = c.score >= least;
          }
          const unsigned all = __ballot_sync(0xffffffffu, reaches);
          int at = 0;
          if (lane == 0 && all != 0) at = atomicAdd(&s_count, __popc(all));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << lane) - 1));
          if (reaches && at < BS_COLLECT) s_got[at] = c;
          if (all != 0xffffffffu) break;
        }
      }
    } else if (tid == 0) {
      s_count = BS_COLLECT + 1;
    }
    __syncthreads();
    // most lists are short of it and some hold much: the bound again, of what they hold
    const int held = s_count;
    if (held > BP_RANKED && held <= BS_COLLECT) {
      uint32_t mine[MOST];
#pragma unroll
      for (int i = 0; i < MOST; ++i) mine[i] = tid + i * BP_THREADS < held ? ordered(static_cast<float>(s_got[tid + i * BP_THREADS].score)) : 0u;
      if (tid < 32) s_tally[tid] = 0;
      if (tid == 0) {
        s_low = 0xffffffffu;
        s_high = s_count = 0;
      }
      __syncthreads();
      least = below(reached(mine, K + 1, K + 16));
      constexpr int KEPT = BS_COLLECT / BP_THREADS;
      Candidate kept[KEPT];
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (tid + i * BP_THREADS < held) kept[i] = s_got[tid + i * BP_THREADS];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (tid + i * BP_THREADS < held && kept[i].score >= least) s_got[atomicAdd(&s_count, 1)] = kept[i];
    }
  }
  __syncthreads();
  const int got = s_count, best = min(got, K + 1);
  auto rank_all = [&]() {
    for (int i = tid; i < got; i += BP_THREADS) {
      const Candidate mine = s_got[i];
      int rank = 0;
#pragma unroll 4
      for (int k = 0; k < got; ++k) {
        const double other = s_got[k].score;
        rank += other > mine.score || (other == mine.score && before(s_got[k], mine)) ? 1 : 0;
      }
      if (rank < K + 1) s_best[rank] = mine;
    }
    __syncthreads();
  };
  // More than can be ranked at once (equal scores, or a few long lists): the K + 1 best one after the other.
  auto one_by_one = [&]() {
    Candidate last{INFINITY, 0.f, -1, -2};
    for (int k = 0; k < best; ++k) {
      Candidate mine{-INFINITY, 0.f, BS_MAX_BEAMS, 0x7fffffff};
      for (int g = tid; g < lists * K; g += BP_THREADS) {
        const int b = beam_of(g / K);
        const uint64_t key = key_at(b, g / K, g % K);
        if (key == 0) continue;
        const Candidate c = candidate(b, key);
        if (before(last, c) && before(c, mine)) mine = c;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Candidate other{__shfl_xor_sync(0xffffffffu, mine.score, o), __shfl_xor_sync(0xffffffffu, mine.x, o), __shfl_xor_sync(0xffffffffu, mine.beam, o),
                              __shfl_xor_sync(0xffffffffu, mine.token, o)};
        if (before(other, mine)) mine = other;
      }
      if (lane == 0) s_got[warp] = mine;
      __syncthreads();
      last = s_got[0];
      for (int w = 1; w < WARPS; ++w)
        if (before(s_got[w], last)) last = s_got[w];
      if (tid == 0) s_best[k] = last;
      __syncthreads();
    }
  };
  const bool many = got > BS_COLLECT;
  if (many) one_by_one();
  else rank_all();
  // ---- continuations of different beams that are too near each other: those beams' sums in 64 bits ----
  if (tid + 1 < best) {
    const Candidate &c = s_best[tid], &d = s_best[tid + 1];
    if (c.beam != d.beam && c.score - d.score <= BS_NEAR && (s_kind[c.beam] == 2 || s_kind[d.beam] == 2)) s_again[c.beam] = s_again[d.beam] = s_any = 1;
  }
  __syncthreads();
  if (s_any) {
    for (int b = 0; b < B; ++b) {
      if (!s_again[b] || s_kind[b] != 2) continue;
      const T* p = static_cast<const T*>(s.logits) + (row0 + b) * s.ld;
      const double top = s_ref[b] * LN2_64;
      double all = 0.0;
#pragma unroll 4
      for (int i = tid; i < s.vocab; i += BP_THREADS) all += exp(static_cast<double>(Logits<T>::one(p + i)) - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (lane == 0) s_sum[warp] = all;
      __syncthreads();
      if (tid == 0) {
        all = 0.0;
        for (int w = 0; w < WARPS; ++w) all += s_sum[w];
        s_total[b] = top + log(all);
      }
      __syncthreads();
    }
    if (many) {
      one_by_one();
    } else {
      for (int i = tid; i < got; i += BP_THREADS)
        if (s_kind[s_got[i].beam] == 2) s_got[i].score = s_score[s_got[i].beam] + (static_cast<double>(s_got[i].x) - s_total[s_got[i].beam]);
      __syncthreads();
      rank_all();
    }
  }
  if (tid < K) {
    const bool there = tid < best && s_best[tid].score > -INFINITY;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * K + tid;
    a.scores[at] = there ? static_cast<float>(s_best[tid].score) : -INFINITY;
    a.parents[at] = there ? s_best[tid].beam : -1;
    a.tokens[at] = there ? s_best[tid].token : -1;
    a.finished[at] = there && (s_kind[s_best[tid].beam] == 1 || (a.eos >= 0 && s_best[tid].token == a.eos)) ? 1 : 0;
  }
}

// ---------------------------------------------------------------------------
// beam_tables_kernel, beam_move_kernel
//
// Row b of a request becomes a child of its row p = parents[b].  Its table is the parent's; a block that is full is shared.  The open
// block, which the next tokens go to, stays with the first row that has it, and the others get a copy in a block from the stack.  A block that no
// row has any more goes onto the stack.
//
// beam_tables_kernel: a CTA per request; a thread per column of its tables (a row's neighbours are the next thread's, so that the loads are whole
// lines).  Rows with children hold their blocks; only the blocks of rows without have to be looked for among those (mostly the first looked
// at has it: a prompt's block).  It leaves the request's copies and given-back blocks in lists, since their places on the stack depend on the requests before.  Further
// CTAs bring the histories.
// beam_move_kernel: every CTA forms the prefix sums over the requests' lists, and then does its share of the copies (pieces of 4 KB, a warp
// each), of the new entries and of the stack.
//
// Bound: latency for one request; HBM for the copies (every copied token read and written once in all planes) and the histories.
// ---------------------------------------------------------------------------
constexpr int BR_THREADS = 256, BR_MAX_ROWS = 8192, BR_PIECE = 4096, BR_HISTORY = 1024;

struct ReorderArgs {
  const int32_t* parents;
  int n, beams;
  const int32_t* tables;
  int64_t bt_stride;
  int bt_width, block_size, num_blocks;
  const int32_t *lens, *first;
  int32_t* free_blocks;
  int capacity;
  const int32_t* num_free;
  unsigned char* cache;
  int planes;
  int64_t plane_bytes, token_bytes;
  const int64_t* history;
  int64_t history_stride;
  int history_width;
  const int32_t* history_lens;
  const int64_t* tokens;
  int32_t *tables_out, *lens_out, *num_free_out;
  int64_t* history_out;
  int32_t* history_lens_out;
  int2* counts;   // [n] copies, given-back blocks
  int4* copies;   // [n][beams] row, block, column, tokens
  int32_t* given;  // [n][beams * bt_width] by column and row
};

__global__ void __launch_bounds__(BR_THREADS) beam_tables_kernel(const ReorderArgs a) {
  __shared__ int s_p[32], s_len[32], s_have[32], s_need[32], s_first[32], s_open[32];
  __shared__ int s_x[32][BR_THREADS];
  __shared__ int s_warp[BR_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.beams, W = a.bt_width, bs = a.block_size;
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  if (static_cast<int>(blockIdx.x) >= a.n) {
    // ---- histories: pieces of rows ----
    const int pieces = max(1, (a.history_width + BR_HISTORY - 1) / BR_HISTORY);
    const int64_t all = static_cast<int64_t>(a.n) * B * pieces;
    for (int64_t u = blockIdx.x - a.n; u < all; u += gridDim.x - a.n) {
      const int row = static_cast<int>(u / pieces), j0 = static_cast<int>(u - static_cast<int64_t>(row) * pieces) * BR_HISTORY;
      const int p = __ldg(a.parents + row);
      const bool alive = p >= 0 && p < B;
      const int from = row / B * B + (alive ? p : 0);
      const int said = alive ? min(max(0, __ldg(a.history_lens + from)), a.history_width) : 0;
      const int64_t token = a.tokens != nullptr && alive ? __ldg(reinterpret_cast<const long long*>(a.tokens) + row) : -1;
      const int64_t *in = a.history + from * a.history_stride;
      int64_t* out = a.history_out + static_cast<int64_t>(row) * a.history_width;
      const int j1 = min(a.history_width, j0 + BR_HISTORY);
#pragma unroll
      for (int e = 0; e < BR_HISTORY / BR_THREADS; ++e) {
        const int j = j0 + e * BR_THREADS + tid;
        if (j < j1) out[j] = j < said ? __ldg(reinterpret_cast<const long long*>(in) + j) : j == said ? token : -1;
      }
      if (j0 == 0 && tid == 0) a.history_lens_out[row] = said + (token >= 0 && said < a.history_width ? 1 : 0);
    }
    return;
  }
  const int r = blockIdx.x, row0 = r * B;
  const int64_t full = static_cast<int64_t>(W) * bs;
  auto old = [&](int q, int j) {
    const int x = __ldg(a.tables + static_cast<int64_t>(row0 + q) * a.bt_stride + j);
    return x >= 0 && x < a.num_blocks ? x : -1;
  };
  if (tid < B) {
    const int p = __ldg(a.parents + row0 + tid), len = __ldg(a.lens + row0 + tid);
    s_p[tid] = p >= 0 && p < B ? p : -1;
    s_len[tid] = len >= 0 && len <= full ? len : 0;
    s_have[tid] = (s_len[tid] + bs - 1) / bs;
    s_first[tid] = min(a.first != nullptr ? max(0, __ldg(a.first + r)) : 0, s_len[tid] / bs);
  }
  __syncthreads();
  if (warp == 0) {
    // ---- open blocks ----
    const int p = lane < B ? s_p[lane] : -1, len = p >= 0 ? s_len[p] : 0, column = len / bs;
    const int mine = len % bs > 0 ? old(p, column) : -1;
    bool copied = false;
    for (int b = 0; b < B; ++b) {
      const int q = s_p[b];
      if (mine >= 0 && b < lane && q >= 0 && column < s_have[q] && (q == p || old(q, column) == mine)) copied = true;
    }
    const unsigned copies = __ballot_sync(0xffffffffu, copied);
    if (lane < B) {
      s_need[lane] = p >= 0 ? s_have[p] : 0;
      s_open[lane] = copied ? column : -1;
      a.lens_out[row0 + lane] = len;
      if (copied) a.copies[static_cast<int64_t>(row0) + __popc(copies & ((1u << lane) - 1))] = make_int4(lane, mine, column, len - column * bs);
    }
    if (lane == 0) a.counts[r].x = __popc(copies);
  }
  __syncthreads();
  // ---- the tables, column by column ----
  int before = 0;
  for (int j0 = 0; j0 < W; j0 += BR_THREADS) {
    const int j = j0 + tid;
    unsigned gone = 0;
    if (j < W) {
#pragma unroll 4
      for (int q = 0; q < B; ++q) s_x[q][tid] = j < s_have[q] ? old(q, j) : -1;
      unsigned held = 0;  // rows whose block some child has
      for (int b = 0; b < B; ++b) {
        const int p = s_p[b];
        const bool has = j < s_need[b] && j != s_open[b];
        if (has) held |= 1u << p;
        a.tables_out[static_cast<int64_t>(row0 + b) * W + j] = has ? s_x[p][tid] : -1;
      }
      for (int q = 0; q < B; ++q) {
        const int x = s_x[q][tid];
        if (x < 0 || j < s_first[q] || ((held >> q) & 1)) continue;
        bool kept = false;
        for (unsigned m = held; m != 0 && !kept; m &= m - 1) kept = s_x[__ffs(m) - 1][tid] == x;
        for (unsigned m = gone; m != 0 && !kept; m &= m - 1) kept = s_x[__ffs(m) - 1][tid] == x;
        if (!kept) gone |= 1u << q;
      }
    }
    const int mine = __popc(gone);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int at = before + incl - mine;
    for (int w = 0; w < BR_THREADS / 32; ++w) {
      if (w < warp) at += s_warp[w];
      before += s_warp[w];
    }
    int32_t* out = a.given + static_cast<int64_t>(row0) * W + at;
    for (unsigned m = gone; m != 0; m &= m - 1) *out++ = s_x[__ffs(m) - 1][tid];
    __syncthreads();
  }
  if (tid == 0) a.counts[r].y = before;
}

__global__ void __launch_bounds__(BR_THREADS) beam_move_kernel(const ReorderArgs a) {
  extern __shared__ int s_sums[];  // copies and given-back blocks before each request
  int *const s_take = s_sums, *const s_back = s_sums + a.n + 1;
  __shared__ int s_warp[BR_THREADS / 32][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n, W = a.bt_width, bs = a.block_size;
  b2::pdl_wait();
  {
    const int per = (n + BR_THREADS - 1) / BR_THREADS, r0 = min(n, tid * per), r1 = min(n, r0 + per);
    int x = 0, y = 0;
    for (int r = r0; r < r1; ++r) {
      const int2 c = a.counts[r];
      s_take[r] = c.x;
      s_back[r] = c.y;
      x += c.x;
      y += c.y;
    }
    int ix = x, iy = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ux = __shfl_up_sync(0xffffffffu, ix, o), uy = __shfl_up_sync(0xffffffffu, iy, o);
      if (lane >= o) {
        ix += ux;
        iy += uy;
      }
    }
    if (lane == 31) {
      s_warp[warp][0] = ix;
      s_warp[warp][1] = iy;
    }
    __syncthreads();
    int bx = ix - x, by = iy - y;
    for (int w = 0; w < warp; ++w) {
      bx += s_warp[w][0];
      by += s_warp[w][1];
    }
    for (int r = r0; r < r1; ++r) {
      const int cx = s_take[r], cy = s_back[r];
      s_take[r] = bx;
      s_back[r] = by;
      bx += cx;
      by += cy;
    }
    if (tid == BR_THREADS - 1) {
      s_take[n] = bx;
      s_back[n] = by;
    }
    __syncthreads();
  }
  const int take = s_take[n], back = s_back[n], height = max(0, min(__ldg(a.num_free), a.capacity)), top = height + back, left = min(a.capacity, max(0, top - take));
  auto request_of = [&](const int* sums, int i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sums[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  auto returned = [&](int k) {
    const int r = request_of(s_back, k);
    return a.given[static_cast<int64_t>(r) * a.beams * W + k - s_back[r]];
  };
  // copy c goes to the block at place top - 1 - c of the stack with the given-back blocks on it
  auto block_for = [&](int c) {
    const int at = top - 1 - c;
    if (at < 0) return -1;
    const int x = at < height ? a.free_blocks[at] : returned(at - height);
    return x >= 0 && x < a.num_blocks ? x : -1;
  };
  const int first = blockIdx.x * BR_THREADS + tid, step = gridDim.x * BR_THREADS;
  for (int c = first; c < take; c += step) {
    const int r = request_of(s_take, c);
    const int4 copy = a.copies[static_cast<int64_t>(r) * a.beams + c - s_take[r]];
    const int block = block_for(c);
    const int64_t row = static_cast<int64_t>(r) * a.beams + copy.x;
    a.tables_out[row * W + copy.z] = block;
    if (block < 0) a.lens_out[row] = copy.z * bs;
  }
  for (int i = height + first; i < left; i += step) a.free_blocks[i] = returned(i - height);
  if (first == 0) *a.num_free_out = left;
  // ---- the cache ----
  const int64_t block_bytes = bs * a.token_bytes;
  const int pieces = static_cast<int>((block_bytes + BR_PIECE - 1) / BR_PIECE);
  const int64_t per_copy = static_cast<int64_t>(a.planes) * pieces, units = take * per_copy;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (BR_THREADS / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (BR_THREADS / 32) + warp; u < units; u += warps) {
    const int c = static_cast<int>(u / per_copy), rest = static_cast<int>(u - c * per_copy), plane = rest / pieces, piece = rest - plane * pieces;
    const int r = request_of(s_take, c);
    const int4 copy = a.copies[static_cast<int64_t>(r) * a.beams + c - s_take[r]];
    const int64_t bytes = copy.w * a.token_bytes, from = static_cast<int64_t>(piece) * BR_PIECE;
    if (from >= bytes) continue;
    const int block = block_for(c);
    if (block < 0) continue;
    const uint4* src = reinterpret_cast<const uint4*>(a.cache + plane * a.plane_bytes + copy.y * block_bytes + from);
    uint4* dst = reinterpret_cast<uint4*>(a.cache + plane * a.plane_bytes + block * block_bytes + from);
    const int vectors = static_cast<int>(min(static_cast<int64_t>(BR_PIECE), bytes - from) / 16);
    uint4 v[BR_PIECE / 512];
#pragma unroll
    for (int e = 0; e < BR_PIECE / 512; ++e)
      if (e * 32 + lane < vectors) v[e] = src[e * 32 + lane];
#pragma unroll
    for (int e = 0; e < BR_PIECE / 512; ++e)
      if (e * 32 + lane < vectors) dst[e * 32 + lane] = v[e];
  }
  b2::pdl_release_results();  // later kernels may read the lengths and tables ahead of their dependency wait
}

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    B2_CUDA(cudaFuncSetAttribute(beam_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (BR_MAX_ROWS + 1) * static_cast<int>(sizeof(int))));
    done[dev].store(true, std::memory_order_release);
  }
  return B2_OK;
}

struct SelectPlan {
  int tiles, grid, parts, capacity;
  int64_t keys_bytes, bytes;
};
SelectPlan plan_select(int num_sms, int rows, int vocab, int picks, bool fp32) {
  SelectPlan p;
  // (a row may begin anywhere between two 16-byte boundaries)
  const int64_t size = fp32 ? 4 : 2, chunks = (vocab * size + 16 - size + 15) / 16;
  p.tiles = static_cast<int>(std::max<int64_t>(1, (chunks * 16 + BS_TILE_BYTES - 1) / BS_TILE_BYTES));
  const int64_t total = static_cast<int64_t>(rows) * p.tiles;
  p.grid = static_cast<int>(std::min<int64_t>(total, static_cast<int64_t>(num_sms) * BS_CTAS_PER_SM));
  const int64_t least = total / std::max(1, p.grid);  // tiles of the shortest range
  p.parts = static_cast<int>(std::min<int64_t>(p.tiles, (p.tiles + least - 1) / std::max<int64_t>(1, least) + 1));
  p.capacity = picks * (fp32 ? 4 : 8) * BS_VECTORS + 256;  // (K threads' logits reach the bound of a first tile, or more where they are equal)
  p.keys_bytes = (static_cast<int64_t>(rows) * p.parts * picks * 8 + 15) / 16 * 16;
  p.bytes = p.keys_bytes + static_cast<int64_t>(rows) * p.parts * static_cast<int64_t>(sizeof(double2));
  return p;
}

}  // namespace

extern "C" {

int64_t b2_beam_select_workspace(b2_ctx* ctx, int n, int beams, int vocab, int picks, int fp32) {
  if (ctx == nullptr || n < 0 || beams < 1 || beams > BS_MAX_BEAMS || picks < 1 || picks > BS_MAX_PICKS || vocab < 1 || static_cast<int64_t>(n) * beams > 1 << 24) return -1;
  return n == 0 ? 0 : plan_select(ctx->num_sms, n * beams, vocab, picks, fp32 != 0).bytes;
}

int b2_beam_select(b2_ctx* ctx, const void* logits, int64_t ld, int fp32, int n, int beams, int vocab, const float* scores, const uint8_t* finished, int picks, int eos_token,
                   float* scores_out, int32_t* parents_out, int64_t* tokens_out, uint8_t* finished_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n < 0) return B2_ERR_ARG;
  if (n == 0) return B2_OK;
  const int64_t need = b2_beam_select_workspace(ctx, n, beams, vocab, picks, fp32);
  if (need < 0) return b2::set_error(B2_ERR_SHAPE, "%d requests of %d beams, %d picks of %d: at most %d beams and %d picks", n, beams, picks, vocab, BS_MAX_BEAMS, BS_MAX_PICKS);
  const int64_t row_tiles = (static_cast<int64_t>(vocab) * (fp32 ? 4 : 2) + 30) / BS_TILE_BYTES + 1;
  if (row_tiles * n * beams >= 1ll << 31 || static_cast<int64_t>(vocab) + BS_TILE_BYTES >= 1ll << 31)
    return b2::set_error(B2_ERR_SHAPE, "%d rows of %d tokens", n * beams, vocab);
  if (!logits || !scores || !scores_out || !parents_out || !tokens_out || !finished_out || ld < vocab) return B2_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) return B2_ERR_ARG;
  const SelectPlan p = plan_select(ctx->num_sms, n * beams, vocab, picks, fp32 != 0);
  char* ws = static_cast<char*>(workspace);
  const ScanArgs s{logits, ld, n * beams, beams, vocab, picks, p.tiles, p.parts, p.capacity, scores, finished, reinterpret_cast<uint64_t*>(ws),
                   reinterpret_cast<double2*>(ws + p.keys_bytes)};
  const PickArgs k{s, p.grid, eos_token, scores_out, parents_out, tokens_out, finished_out};
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  const size_t smem = static_cast<size_t>(p.capacity) * 8;
  B2_CUDA(b2_launch(fp32 ? beam_scan_kernel<float> : beam_scan_kernel<__nv_bfloat16>, dim3(p.grid), dim3(BS_THREADS), smem, on, s));
  B2_CUDA(b2_launch(fp32 ? beam_pick_kernel<float> : beam_pick_kernel<__nv_bfloat16>, dim3(n), dim3(BP_THREADS), 0, on, k));
  return B2_OK;
}

int64_t b2_reorder_beams_workspace(int n, int beams, int bt_width) {
  if (n < 0 || beams < 1 || beams > 32 || bt_width < 0 || static_cast<int64_t>(n) * beams > BR_MAX_ROWS) return -1;
  const int64_t rows = static_cast<int64_t>(n) * beams;
  return rows * sizeof(int4) + (n * static_cast<int64_t>(sizeof(int2)) + 15) / 16 * 16 + rows * bt_width * 4;
}

int b2_reorder_beams(b2_ctx* ctx, const int32_t* parents, int n, int beams, const int32_t* block_tables, int64_t bt_stride, int bt_width, const int32_t* context_lens,
                     const int32_t* first_blocks, int32_t* free_blocks, int free_capacity, const int32_t* num_free, int block_size, void* cache, int planes,
                     int64_t plane_bytes, int num_blocks, int64_t token_bytes, const int64_t* history, int64_t history_stride, int history_width,
                     const int32_t* history_lens, const int64_t* tokens, int32_t* tables_out, int32_t* lens_out, int32_t* num_free_out, int64_t* history_out,
                     int32_t* history_lens_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n < 0 || free_capacity < 0 || block_size <= 0 || planes < 0 || num_blocks <= 0 || token_bytes <= 0 || history_width < 0) return B2_ERR_ARG;
  const int64_t need = b2_reorder_beams_workspace(n, beams, bt_width);
  if (need < 0) return b2::set_error(B2_ERR_SHAPE, "%d requests of %d beams: at most 32 beams and %d rows", n, beams, BR_MAX_ROWS);
  if (n > 0 && (bt_width <= 0 || bt_stride < bt_width || !parents || !block_tables || !context_lens || !tables_out || !lens_out)) return B2_ERR_ARG;
  if (!num_free || !num_free_out || (free_capacity > 0 && !free_blocks) || (planes > 0 && !cache)) return B2_ERR_ARG;
  if (history != nullptr && (!history_lens || !history_out || !history_lens_out || history_stride < history_width)) return B2_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(cache) | token_bytes | (planes > 1 ? plane_bytes : 0)) & 15) return B2_ERR_ARG;
  constexpr int64_t limit = (1ll << 31) - 1;
  if (static_cast<int64_t>(n) * beams * bt_width > limit / block_size || static_cast<int64_t>(n) * beams * bt_width + free_capacity > limit || num_blocks > limit / block_size ||
      token_bytes > limit || block_size * token_bytes > limit || planes > 65536 || planes * ((block_size * token_bytes + BR_PIECE - 1) / BR_PIECE) > limit)
    return b2::set_error(B2_ERR_SHAPE, "tokens, blocks and pieces of a copy must each add up to less than 2^31");
  if ((n > 0 && workspace == nullptr) || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) return B2_ERR_ARG;
  const int rc = configure_once();
  if (rc != B2_OK) return rc;
  const int64_t rows = static_cast<int64_t>(n) * beams;
  char* ws = static_cast<char*>(workspace);
  const int64_t counts_bytes = (n * static_cast<int64_t>(sizeof(int2)) + 15) / 16 * 16;
  const ReorderArgs a{parents, n, beams, block_tables, bt_stride, bt_width, block_size, num_blocks, context_lens, first_blocks, free_blocks, free_capacity, num_free,
                      static_cast<unsigned char*>(cache), planes, plane_bytes, token_bytes, history, history_stride, history != nullptr ? history_width : 0, history_lens, tokens,
                      tables_out, lens_out, num_free_out, history_out, history_lens_out, reinterpret_cast<int2*>(ws + rows * sizeof(int4)), reinterpret_cast<int4*>(ws),
                      reinterpret_cast<int32_t*>(ws + rows * sizeof(int4) + counts_bytes)};
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  // histories: a CTA for each piece of a row, four per SM at most
  const int64_t pieces = history != nullptr ? rows * std::max(1, (history_width + BR_HISTORY - 1) / BR_HISTORY) : 0;
  const int more = static_cast<int>(std::min<int64_t>(pieces, 4 * ctx->num_sms));
  if (n + more > 0) B2_CUDA(b2_launch(beam_tables_kernel, dim3(n + more), dim3(BR_THREADS), 0, on, a));
  const int64_t most = rows * planes * ((block_size * token_bytes + BR_PIECE - 1) / BR_PIECE) / (BR_THREADS / 32);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4 * ctx->num_sms, most)));
  B2_CUDA(b2_launch(beam_move_kernel, dim3(grid), dim3(BR_THREADS), 2 * (n + 1) * sizeof(int), on, a));
  return B2_OK;
}

}  // extern "C"
