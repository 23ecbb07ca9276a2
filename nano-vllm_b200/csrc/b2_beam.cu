// A step of beam search: the best continuations of each request, and what its beams have in the cache following them.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// beam_scan_kernel, beam_pick_kernel
//
// A continuation of beam b by token v has the score s_b + x_bv - log sum_u exp x_bu.  One pass over the logits gives the sums, and the largest
// logit of each chunk of 2 KB.  With those, the K best are in at most K chunks: a chunk that K others have a larger maximum than (or the same, and
// lie before it) holds none of them.  So the second kernel reads 2 KB for each of about K maxima, and the first does nothing for the selection but to store
// the maxima.  (Before, the first kernel kept a list of candidates with a rising bound: 33 instructions a logit and threads of a warp that had parted, 53 us
// for 64 requests of 8 beams over 151936 tokens.)
//
// beam_scan_kernel: the chunks of all rows are dealt to the warps in contiguous equal ranges, so that every SM streams whatever the batch; warps have
// nothing to do with each other.  Exponentials of the hardware, sums of a thread's 32 or 16 logits of a chunk in 32 bits, and of those in 64.
//
// beam_pick_kernel: a CTA per request.  Scores are formed in 64 bits.  The sums' error could turn the order of continuations of two beams that lie
// closer than BS_NEAR.  Each is off by 2^-22 (2.4e-7) of an exponential, 2^-20 log(2) (6.6e-7) of an exponent's rounding, which is below 32 (BS_ABOVE; what lies further down than that weighs less than 2^-14
// even over 2^18 tokens), 3e-7 of log2(e) in 24 bits there, and ten additions in 32 bits (6e-7): 1.8e-6, 3.6e-6 for the two.  Where two of those that may be among the K best are that near, their beams'
// sums are formed again in 64 bits from the logits, in an order and with a reference that depend on nothing but the row.
//
// Bound: the pass by HBM and the exponentials' unit, 31 us for 64 requests of 8 beams over 151936 tokens (60 % and 69 %); what follows by its chain of steps, 11 us there.
// ---------------------------------------------------------------------------
constexpr int BS_THREADS = 128, BS_VECTORS = 4, BS_CTAS_PER_SM = 8, BS_WARPS = BS_THREADS / 32;
constexpr int BS_CHUNK_BYTES = 32 * BS_VECTORS * 16;
constexpr int BS_MAX_PICKS = 64, BS_MAX_BEAMS = 32;
constexpr int BP_THREADS = 512, BP_WARPS = BP_THREADS / 32;
constexpr int BP_CHUNKS = 512, BP_COLLECT = 1536;  // chunks and candidates that a request looks at
constexpr double BS_NEAR = 4e-6;
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LOG2E_64 = 1.4426950408889634, LN2_64 = 0.6931471805599453;
constexpr float BS_PLAIN = 65536.f;  // below this size x log2(e) is formed in 32 bits
constexpr float BS_ABOVE = 22.f;     // the sum's reference is raised when a logit is this far above it: exponents stay below 32, whose last bit is 2^-19

struct ScanArgs {
  const void* logits;
  int64_t ld;
  int rows, beams, vocab, picks;
  int chunks, parts, warps;  // of a row: chunks, most parts; of the scan: warps
  const float* scores;
  const uint8_t* finished;
  float* maxima;   // [rows][chunks]
  double2* sums;   // [rows][parts] (M, sum of 2^(x log2(e) - M)); M is a whole number, -inf where there is nothing
};

__device__ __forceinline__ uint32_t ordered(float x) {  // unsigned order = order of the numbers; -0 is 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }
// 2^x of a whole number x <= 0, exactly; 0 below the normal range (and for NaN, the difference of two -inf)
__device__ __forceinline__ double power_of_two(double x) { return x > -1023.0 ? __longlong_as_double(static_cast<long long>(1023 + static_cast<int>(x)) << 52) : 0.0; }

// NaN counts as -inf, +inf as the type's largest number
template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
  static __device__ __forceinline__ float one(const float* p) { return clean(__ldg(p)); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float largest(const uint4 (&v)[BS_VECTORS]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)), fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
    return m;
  }
};
template <>
struct Logits<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), b2::bf16_hi(0x7f7f0000u)); }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return clean(__uint_as_float(static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(p))) << 16)); }
  static __device__ __forceinline__ uint32_t max2(uint32_t x, uint32_t y) {
    const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) { b2::unpack8(v, f); }
  static __device__ __forceinline__ float largest(const uint4 (&v)[BS_VECTORS]) {
    uint32_t w = 0xff80ff80u;
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i) w = max2(w, max2(max2(v[i].x, v[i].y), max2(v[i].z, v[i].w)));
    return fmaxf(fmaxf(b2::bf16_lo(w), b2::bf16_hi(w)), -INFINITY);
  }
};

// A row begins anywhere; its chunks are counted from the 16-byte boundary at or before it.
template <typename T>
struct Row {
  static constexpr int N = Logits<T>::N, CHUNK = BS_CHUNK_BYTES / static_cast<int>(sizeof(T));
  const T* p;
  int vocab, shift;
  __device__ __forceinline__ Row(const ScanArgs& a, int row) : p(static_cast<const T*>(a.logits) + row * a.ld), vocab(a.vocab) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  }
  // the token of element 0 of lane `lane`'s vector i; may lie before or behind the row
  __device__ __forceinline__ int token(int chunk, int i, int lane) const { return chunk * CHUNK - shift + (i * 32 + lane) * N; }
  // (by value: an array would go through memory, and a load would be waited for as soon as it is made)
  static __device__ __noinline__ uint4 edge(const T* p, int vocab, int first) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (N == 8) {
        const int t = first + 2 * k;
        const uint32_t lo = t >= 0 && t < vocab ? __ldg(reinterpret_cast<const unsigned short*>(p) + t) : 0xff80u;
        const uint32_t hi = t + 1 >= 0 && t + 1 < vocab ? __ldg(reinterpret_cast<const unsigned short*>(p) + t + 1) : 0xff80u;
        w[k] = lo | hi << 16;
      } else {
        const int t = first + k;
        w[k] = t >= 0 && t < vocab ? __float_as_uint(__ldg(reinterpret_cast<const float*>(p) + t)) : 0xff800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // a lane's vectors of a chunk, -inf in the places that are not the row's
  __device__ __forceinline__ void load(int chunk, int lane, uint4 (&v)[BS_VECTORS]) const {
    const int first = chunk * CHUNK - shift;
    if (first >= 0 && first + CHUNK <= vocab) {
      const uint4* q = reinterpret_cast<const uint4*>(p + first) + lane;
#pragma unroll
      for (int i = 0; i < BS_VECTORS; ++i) v[i] = __ldg(q + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < BS_VECTORS; ++i) v[i] = edge(p, vocab, token(chunk, i, lane));
    }
  }
  // sum of 2^(x log2(e) - ref) of a lane's logits, in 64 bits; log2(e) is the 24-bit one of the other chunks, which a row's log is put right for as a whole
  __device__ __noinline__ double exact_sum(int chunk, int lane, double ref) const {
    double sum = 0.0;
    for (int i = 0; i < BS_VECTORS * N; ++i) {
      const int t = token(chunk, i / N, lane) + i % N;
      if (t >= 0 && t < vocab) sum += exp2(__dmul_rn(Logits<T>::one(p + t), LOG2E) - ref);
    }
    return sum;
  }
};

// Ranges of `total` chunks: warp x of X
struct ScanDeal {
  int base, rem;
  __device__ __forceinline__ ScanDeal(int total, int X) : base(total / X), rem(total % X) {}
  __device__ __forceinline__ int begin_of(int x) const { return x * base + min(x, rem); }
  __device__ __forceinline__ int owner_of(int t) const {
    const int big = rem * (base + 1);
    return t < big ? t / (base + 1) : rem + (t - big) / base;
  }
};

template <typename T>
__global__ void __launch_bounds__(BS_THREADS, BS_CTAS_PER_SM) beam_scan_kernel(const ScanArgs a) {
  constexpr int N = Logits<T>::N;
  const int lane = threadIdx.x & 31, x = blockIdx.x * BS_WARPS + b2::uniform(static_cast<int>(threadIdx.x >> 5));
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  if (x >= a.warps) return;
  const ScanDeal deal(a.rows * a.chunks, a.warps);
  int u = deal.begin_of(x);
  const int end = deal.begin_of(x + 1);
  while (u < end) {
    const int row = u / a.chunks, c0 = u - row * a.chunks, c1 = min(a.chunks, c0 + end - u);
    u += c1 - c0;
    if (!(a.scores[row] > -INFINITY) || (a.finished != nullptr && a.finished[row] != 0)) continue;  // (it has one continuation or none)
    const Row<T> r(a, row);
    uint4 next[BS_VECTORS];
    r.load(c0, lane, next);
    // The sum's reference is a power of two, so that raising it is exact, and x log2(e) - M is one rounding of an exact product.
    double ref = -INFINITY, sum = 0.0;
    float ref_low = -INFINITY, raise_at = -INFINITY;  // ref as far as 32 bits go; the logit above which it is raised
    auto raise = [&](double to) {
      if (to > ref) {
        sum *= power_of_two(ref - to);
        ref = to;
        ref_low = static_cast<float>(to);
        raise_at = ref_low * (1.f / LOG2E) + BS_ABOVE;
      }
    };
    for (int c = c0; c < c1; ++c) {
      uint4 now[BS_VECTORS];
#pragma unroll
      for (int i = 0; i < BS_VECTORS; ++i) now[i] = next[i];
      if (c + 1 < c1) r.load(c + 1, lane, next);
      // (the same in all lanes from here on, but for the sums)
      const float top = Logits<T>::clean(number_of(__reduce_max_sync(0xffffffffu, ordered(Logits<T>::largest(now)))));
      if (lane == 0) a.maxima[static_cast<int64_t>(row) * a.chunks + c] = top;
      if (top == -INFINITY) continue;
      bool odd = fabsf(top) >= BS_PLAIN;
      if (!odd) {
        if (top > raise_at) raise(rintf(top * LOG2E));
        uint64_t sums[2] = {};
        const uint64_t minus = b2::pair_of(-ref_low, -ref_low), scale = b2::pair_of(LOG2E, LOG2E);
#pragma unroll
        for (int i = 0; i < BS_VECTORS; ++i) {
          float f[N];
          Logits<T>::unpack(now[i], f);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            float y, z;
            b2::fma_pair(y, z, b2::pair_of(f[e], f[e + 1]), scale, minus);
            sums[(e >> 1) & 1] = b2::add_pair(sums[(e >> 1) & 1], b2::pair_of(b2::ex2(y), b2::ex2(z)));
          }
        }
        float y, z;
        b2::halves_of(b2::add_pair(sums[0], sums[1]), y, z);
        odd = __any_sync(0xffffffffu, !(y + z < INFINITY));  // (a NaN among the logits makes the sum one)
        if (!odd) sum += y + z;
      }
      if (odd) {  // infinities, NaN and very large numbers
        raise(rint(__dmul_rn(top, LOG2E)));
        sum += r.exact_sum(c, lane, ref);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // the warp that holds the row's first chunk is the first of its parts
    if (lane == 0) a.sums[static_cast<int64_t>(row) * a.parts + x - deal.owner_of(row * a.chunks)] = make_double2(ref, sum);
  }
}

struct PickArgs {
  ScanArgs scan;
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
  constexpr int N = Logits<T>::N;
  __shared__ double s_top[BS_MAX_BEAMS], s_log[BS_MAX_BEAMS], s_score[BS_MAX_BEAMS], s_sum[BP_WARPS], s_power[64];  // log sum exp x: a row's largest logit, and the log of the rest
  __shared__ int s_kind[BS_MAX_BEAMS], s_again[BS_MAX_BEAMS], s_tally[32], s_count, s_any, s_far, s_reach, s_list[BP_CHUNKS];
  __shared__ uint32_t s_low, s_high;
  __shared__ Candidate s_got[BP_COLLECT], s_best[BS_MAX_PICKS + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = s.beams, K = s.picks, row0 = blockIdx.x * B, C = s.chunks;
  const ScanDeal deal(s.rows * s.chunks, s.warps);
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  // ---- each row's sum; the chunks' maxima are on their way meanwhile ----
  constexpr int MOST = 12;  // of a thread that it keeps
  float highest[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) highest[i] = tid + i * BP_THREADS < B * C ? s.maxima[static_cast<int64_t>(row0) * C + tid + i * BP_THREADS] : -INFINITY;
  if (tid < 32) s_tally[tid] = 0;
  if (tid < B) s_again[tid] = 0;
  if (tid == 0) {
    s_count = s_any = s_far = s_reach = 0;
    s_low = 0xffffffffu;
    s_high = 0;
  }
  __syncthreads();
  for (int b = warp; b < B; b += BP_WARPS) {
    const float score = s.scores[row0 + b];
    const int kind = !(score > -INFINITY) ? 0 : s.finished != nullptr && s.finished[row0 + b] != 0 ? 1 : 2;  // no continuation, itself, all tokens
    double top = -INFINITY, all = 0.0;
    float largest = -INFINITY;
    if (kind == 2) {
      for (int g = lane; g < C; g += 32) largest = fmaxf(largest, s.maxima[static_cast<int64_t>(row0 + b) * C + g]);
      largest = number_of(__reduce_max_sync(0xffffffffu, ordered(largest)));
      const int first = (row0 + b) * C, parts = deal.owner_of(first + C - 1) - deal.owner_of(first) + 1;
      const double2* sums = s.sums + static_cast<int64_t>(row0 + b) * s.parts;
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
    }
    if (lane == 0) {
      s_score[b] = score;
      s_kind[b] = kind;
      s_top[b] = largest;
      // log2(e) has 24 bits in the sum's exponents, which makes them this much too large; what carries the sum lies near M
      s_log[b] = (top - top * (static_cast<double>(LOG2E) * LN2_64 - 1.0)) * LN2_64 - largest + log(all);
      if (kind == 2 && fabsf(largest) >= BS_PLAIN && largest > -INFINITY) s_again[b] = s_far = 1;  // (M has not the bits)
    }
  }
  __syncthreads();
  // ---- a row's sum in 64 bits ----
  // (a multiple of 1 / 64 in the exponent from the table, the rest of at most 1 / 128 by the series: the table-driven exponential of P. T. P. Tang)
  auto sum_again = [&](int b) {
    const T* p = static_cast<const T*>(s.logits) + (row0 + b) * s.ld;
    const double top = s_top[b];  // (not the scan's M: rows that are alike have the same sum, whatever their place)
    double all = 0.0;
#pragma unroll 4
    for (int i = tid; i < s.vocab; i += BP_THREADS) {
      const double t = __dmul_rn(Logits<T>::one(p + i) - top, LOG2E_64), k = rint(t * 64.0), d = (t - k * (1.0 / 64.0)) * LN2_64;
      if (t > -64.0) {
        const int n = static_cast<int>(k);
        all += s_power[n & 63] * __longlong_as_double(static_cast<long long>(1023 + (n >> 6)) << 52) * (1.0 + d * (1.0 + d * (0.5 + d * (1.0 / 6.0 + d * (1.0 / 24.0)))));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) s_sum[warp] = all;
    __syncthreads();
    if (tid == 0) {
      all = 0.0;
      for (int w = 0; w < BP_WARPS; ++w) all += s_sum[w];
      s_log[b] = log(all);
    }
    __syncthreads();
  };
  auto fill_powers = [&]() {
    if (tid < 64) s_power[tid] = exp2(tid / 64.0);
    __syncthreads();
  };
  if (s_far) {
    fill_powers();
    for (int b = 0; b < B; ++b)
      if (s_again[b]) sum_again(b);
  }
  auto score_of = [&](int b, float x) { return s_score[b] + (static_cast<double>(x) - s_top[b] - s_log[b]); };
  // the best score in chunk g of the request, -inf where there is none; a finished beam has one, in its first chunk
  auto chunk_score = [&](int g, float x) -> double {
    const int b = g / C, kind = s_kind[b];
    return kind == 2 ? (x > -INFINITY ? score_of(b, x) : -INFINITY) : kind == 1 && g == b * C ? s_score[b] : -INFINITY;
  };
  auto maximum = [&](int g) {
    const int b = g / C;
    return s_kind[b] == 2 ? s.maxima[static_cast<int64_t>(row0) * C + g] : -INFINITY;
  };
  // a bound in ordered bits, a little lower: what lies as near as the sums' error belongs to it
  auto below = [](uint32_t bits) {
    const double t = fminf(number_of(bits), FLT_MAX);  // (all continuations of a score of +inf are above that)
    return t - 2 * BS_NEAR - 2.4e-7 * fabs(t);
  };
  // All lanes: how many of the lane's continuations in chunk g have a score from `bound` on
  auto count_from = [&](int g, double bound) {
    const int b = g / C;
    if (s_kind[b] == 1) return lane == 0 && s_score[b] >= bound ? 1 : 0;
    uint4 v[BS_VECTORS];
    Row<T>(s, row0 + b).load(g - b * C, lane, v);
    int count = 0;
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i) {
      float x[N];
      Logits<T>::unpack(v[i], x);
#pragma unroll
      for (int e = 0; e < N; ++e) count += score_of(b, Logits<T>::clean(x[e])) >= bound ? 1 : 0;  // (no logit in its place: next to the largest numbers a score is lost)
    }
    return count;
  };
  // All lanes: the continuations in chunk g with a score from `bound` on (and perhaps some a little below) are handed to f.
  auto each = [&](int g, double bound, auto f) {
    const int b = g / C;
    if (s_kind[b] == 1) {
      if (lane == 0) f(Candidate{s_score[b], 0.f, b, -1});
      return;
    }
    const Row<T> r(s, row0 + b);
    uint4 v[BS_VECTORS];
    r.load(g - b * C, lane, v);
    const float x0 = fmaxf(-FLT_MAX, __double2float_rd(bound - s_score[b] + s_log[b] + s_top[b]));  // (what is forbidden is no continuation)
#pragma unroll
    for (int i = 0; i < BS_VECTORS; ++i) {
      float x[N];
      Logits<T>::unpack(v[i], x);
      unsigned some = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) some |= x[e] >= x0 ? 1u << e : 0u;
      for (; some != 0; some &= some - 1) {
        const int e = __ffs(some) - 1;
        float y = x[0];
#pragma unroll
        for (int k = 1; k < N; ++k) y = e == k ? x[k] : y;
        y = Logits<T>::clean(y);
        f(Candidate{score_of(b, y), y, b, r.token(g - b * C, i, lane) + e});
      }
    }
    __syncwarp();
  };

  // ---- a bound that at least K + 1 chunks' maxima reach, and not many more ----
  double least = -INFINITY;
  {
    uint32_t mine[MOST], low = 0xffffffffu, high = 0;
    auto value = [&](int g, float x) {
      const double score = chunk_score(g, x);
      return score > -INFINITY ? ordered(static_cast<float>(score)) : 0u;
    };
    const int n = B * C;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int g = tid + i * BP_THREADS;
      mine[i] = g < n ? value(g, highest[i]) : 0u;
      if (mine[i] != 0) {
        low = min(low, mine[i]);
        high = max(high, mine[i]);
      }
    }
    for (int g = tid + MOST * BP_THREADS; g < n; g += BP_THREADS) {  // (very large vocabularies)
      const uint32_t o = value(g, maximum(g));
      if (o != 0) {
        low = min(low, o);
        high = max(high, o);
      }
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
    // the bits that all of them have in common are the bound's
    const int bits = low >= high ? 0 : 32 - __clz(low ^ high);
    uint32_t reach = bits == 32 || high == 0 ? 0u : low >> bits << bits;
    bool any = false;
    for (int bit = bits - 1; bit >= 0; --bit) {
      const uint32_t c = reach | (1u << bit);
      int count = 0;
#pragma unroll
      for (int i = 0; i < MOST; ++i) count += mine[i] >= c ? 1 : 0;
      for (int g = tid + MOST * BP_THREADS; g < n; g += BP_THREADS) count += value(g, maximum(g)) >= c ? 1 : 0;
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0 && count > 0) atomicAdd(s_tally + bit, count);
      __syncthreads();
      const int all = s_tally[bit];
      if (all < K + 1) continue;
      reach = c;
      any = true;
      if (all <= K + 16) break;
    }
    if (any && reach > 0x00800000u) least = below(reach);
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int g = tid + i * BP_THREADS;
      if (mine[i] != 0 && chunk_score(g, highest[i]) >= least) {
        const int at = atomicAdd(&s_reach, 1);
        if (at < BP_CHUNKS) s_list[at] = g;
      }
    }
    for (int g = tid + MOST * BP_THREADS; g < n; g += BP_THREADS) {
      const double score = chunk_score(g, maximum(g));
      if (score > -INFINITY && score >= least) {
        const int at = atomicAdd(&s_reach, 1);
        if (at < BP_CHUNKS) s_list[at] = g;
      }
    }
  }
  __syncthreads();

  // All threads: the first of what each has, in s_got[0]
  auto first_of_all = [&](Candidate mine) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Candidate other{__shfl_xor_sync(0xffffffffu, mine.score, o), __shfl_xor_sync(0xffffffffu, mine.x, o), __shfl_xor_sync(0xffffffffu, mine.beam, o),
                            __shfl_xor_sync(0xffffffffu, mine.token, o)};
      if (before(other, mine)) mine = other;
    }
    __syncthreads();
    if (lane == 0) s_got[warp] = mine;
    __syncthreads();
    mine = s_got[0];
    for (int w = 1; w < BP_WARPS; ++w)
      if (before(s_got[w], mine)) mine = s_got[w];
    return mine;
  };
  const Candidate nothing{-INFINITY, 0.f, BS_MAX_BEAMS, 0x7fffffff};
  int reach = s_reach;
  bool exact = false;
  if (reach > BP_CHUNKS) {
    // Many chunks with the same maximum: all rows' sums in 64 bits, with which the first K + 1 chunks are sure, one after the other.
    fill_powers();
    for (int b = 0; b < B; ++b)
      if (s_kind[b] == 2 && s_top[b] > -INFINITY) sum_again(b);
    exact = true;
    least = -INFINITY;
    Candidate last{INFINITY, 0.f, -1, -2};
    for (reach = 0; reach < K + 1; ++reach) {
      Candidate mine = nothing;
      for (int g = tid; g < B * C; g += BP_THREADS) {
        const Candidate c{chunk_score(g, maximum(g)), 0.f, g / C, g};
        if (c.score > -INFINITY && before(last, c) && before(c, mine)) mine = c;
      }
      last = first_of_all(mine);
      if (!(last.score > -INFINITY)) break;
      if (tid == 0) s_list[reach] = last.token;
    }
    __syncthreads();
  }
  // ---- their continuations that reach the bound ----
  auto collect = [&]() {
    for (int l = warp; l < reach; l += BP_WARPS)
      each(s_list[l], least, [&](const Candidate& c) {
        const int at = atomicAdd(&s_count, 1);
        if (at < BP_COLLECT) s_got[at] = c;
      });
    __syncthreads();
  };
  collect();
  if (s_count > BP_COLLECT) {
    // Fewer chunks than picks, which give no bound, or chunks that hold many of the best: a bound that at least K + 1 of the continuations reach, bit by bit from their number.
    // (64 picks of 50257 tokens of one beam: 97 us; one after the other, as below, 3.3 ms.)
    if (tid < 32) s_tally[tid] = 0;
    __syncthreads();
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = bound | (1u << bit);
      if (c > s_high + 1) continue;  // (no chunk's largest reaches it)
      if (c < 0x00800000u) break;    // (-inf)
      const double t = fminf(number_of(c), FLT_MAX);
      int count = 0;
      for (int l = warp; l < reach; l += BP_WARPS) count += count_from(s_list[l], t);
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0 && count > 0) atomicAdd(s_tally + bit, count);
      __syncthreads();
      const int all = s_tally[bit];
      if (all < K + 1) continue;
      bound = c;
      if (all <= BP_COLLECT / 4) break;
    }
    if (bound != 0) {
      least = below(bound);
      if (tid == 0) s_count = 0;
      __syncthreads();
      collect();
    }
  }
  const int got = s_count, best = min(got, K + 1);
  const bool many = got > BP_COLLECT;
  auto rank_all = [&]() {
    if (!many) {
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
    } else {
      // more than can be ranked at once and no bound between them (equal logits by the thousand): the K + 1 best one after the other (rows of one number, 151936 tokens: 4 picks of 4 beams 258 us, 64 of
      // 32 beams 4 ms)
      Candidate last{INFINITY, 0.f, -1, -2};
      for (int k = 0; k < best; ++k) {
        Candidate mine = nothing;
        for (int l = warp; l < reach; l += BP_WARPS)
          each(s_list[l], -INFINITY, [&](const Candidate& c) {
            if (before(last, c) && before(c, mine)) mine = c;
          });
        last = first_of_all(mine);
        if (tid == 0) s_best[k] = last;
      }
    }
    __syncthreads();
  };
  rank_all();
  // ---- continuations of different beams that are too near each other: those beams' sums in 64 bits ----
  // Those that may belong to the K best are the ones from BS_NEAR below the K-th on: mostly K or K + 1, neighbours in s_best.
  if (!exact && best > 1) {
    if (many) {
      if (tid < B) s_again[tid] = 1;
      if (tid == 0) s_any = 1;
    } else {
      const double last = s_best[min(best, K) - 1].score - BS_NEAR;
      auto near = [&](const Candidate& c, const Candidate& d) { return c.beam != d.beam && fabs(c.score - d.score) <= BS_NEAR && d.score >= last && (s_kind[c.beam] == 2 || s_kind[d.beam] == 2); };
      if (tid + 1 < best && near(s_best[tid], s_best[tid + 1])) s_again[s_best[tid].beam] = s_again[s_best[tid + 1].beam] = s_any = 1;
      for (int i = tid; i < got; i += BP_THREADS) {
        const Candidate mine = s_got[i];
        if (best <= K || mine.score < last || !before(s_best[K], mine)) continue;
        for (int k = 0; k < got; ++k)
          if (near(mine, s_got[k])) s_again[mine.beam] = s_again[s_got[k].beam] = s_any = 1;
      }
    }
  }
  __syncthreads();
  if (s_any) {
    fill_powers();
    for (int b = 0; b < B; ++b)
      if (s_again[b] && s_kind[b] == 2 && s_top[b] > -INFINITY) sum_again(b);
    if (!many)
      for (int i = tid; i < got; i += BP_THREADS)
        if (s_kind[s_got[i].beam] == 2) s_got[i].score = score_of(s_got[i].beam, s_got[i].x);
    __syncthreads();
    rank_all();
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
// block, which the next tokens go to, stays with the first row that has it, and the others get a copy in a block from the stack; where it is full in another row, which
// would read what the next tokens write over, all of them get a copy.  A block that no row has any more goes onto the stack.
//
// beam_tables_kernel: a CTA per request, 64 to 256 columns of its tables at a time through shared memory; a warp takes a column, a lane a row, and finds the rows
// that have the same block by a match over the warp.  (A thread per column that compared its rows one after the other: 39 us instead of 11 for seven requests of 29 rows over 400 columns; the other way round with two
// rows, 12 us instead of 15 for two requests of two rows over 10000 columns, where the walk over the columns is most of it.)  It
// leaves the request's copies and given-back blocks in lists, since their places on the stack depend on the requests before.  Further CTAs bring the histories.
// beam_move_kernel: every CTA forms the prefix sums over the requests' lists and looks up what is copied where, and then does its share of the copies (pieces of 4 KB, a
// warp each), of the new entries and of the stack.
//
// Bound: latency for one request (11 us for 4 beams, blocks of 256 tokens in 28 layers, of which the copies take 4.3); else the matches (9 us for 64 requests of 8 rows) and the
// copies, every copied token read and written once in all planes: 12 us for 64 x 8 rows in blocks of 16 tokens, 36 layers, 18 MB each way.
// ---------------------------------------------------------------------------
constexpr int BR_THREADS = 256, BR_WARPS = BR_THREADS / 32, BR_MAX_ROWS = 8192, BR_PIECE = 4096, BR_HISTORY = 1024, BR_COPIES = 1024;
constexpr int BT_THREADS = 512, BT_WARPS = BT_THREADS / 32, BT_COLUMNS = 256, BT_ENTRIES = 32 * (64 + 1);  // (8 rows of 257 and 16 of 129 are fewer)

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

__global__ void __launch_bounds__(BT_THREADS) beam_tables_kernel(const ReorderArgs a) {
  __shared__ int s_p[32], s_len[32], s_have[32], s_need[32], s_first[32], s_open[32];
  __shared__ int s_x[BT_ENTRIES], s_new[BT_ENTRIES];  // [rows][columns + 1] (a column's rows in as many banks)
  __shared__ unsigned s_gone[BT_COLUMNS];  // rows whose block no row has any more
  __shared__ int s_at[BT_COLUMNS];
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
      const int64_t token = a.tokens != nullptr && alive ? max(-1ll, __ldg(reinterpret_cast<const long long*>(a.tokens) + row)) : -1;  // (negative: none)
      const int64_t *in = a.history + from * a.history_stride;
      int64_t* out = a.history_out + static_cast<int64_t>(row) * a.history_width;
      const int j1 = min(a.history_width, j0 + BR_HISTORY);
#pragma unroll
      for (int e = 0; e < BR_HISTORY / BT_THREADS; ++e) {
        const int j = j0 + e * BT_THREADS + tid;
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
  // ---- open blocks: what each row's parent has in the columns in which the rows' lengths end ----
  for (int i = tid; i < B * B; i += BT_THREADS) {
    const int b = i / B, c = i - b * B, p = s_p[b], of = s_p[c], column = of >= 0 ? s_len[of] / bs : 0;
    s_x[i] = p >= 0 && of >= 0 && s_len[of] % bs > 0 && column < s_have[p] ? old(p, column) : -1;
  }
  __syncthreads();
  if (warp == 0) {
    const int p = lane < B ? s_p[lane] : -1, len = p >= 0 ? s_len[p] : 0, column = len / bs;
    const int mine = lane < B ? s_x[lane * B + lane] : -1;
    bool copied = false;  // a row before has the block as well, or any row as a full one
    const int64_t end = (column + 1ll) * bs;
#pragma unroll 4
    for (int b = 0; b < B; ++b) {
      const int other = __shfl_sync(0xffffffffu, len, b);
      copied = copied || (lane < B && mine >= 0 && s_x[b * B + lane] == mine && (b < lane || other >= end));
    }
    __syncwarp();
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
  // ---- the tables ----
  const int p = lane < B ? s_p[lane] : -1, have = lane < B ? s_have[lane] : 0, need = lane < B ? s_need[lane] : 0, own_first = lane < B ? s_first[lane] : 0,
            open = lane < B ? s_open[lane] : -1;
  const int shift = B <= 8 ? 8 : B <= 16 ? 7 : 6, most = 1 << shift, line = most + 1;  // columns at a time
  int before = 0;
  for (int j0 = 0; j0 < W; j0 += most) {
    const int columns = min(most, W - j0);
#pragma unroll 4
    for (int i = tid; i < B << shift; i += BT_THREADS) {
      const int q = i >> shift, c = i & (most - 1);
      s_x[q * line + c] = j0 + c < s_have[q] ? old(q, j0 + c) : -1;
    }
    __syncthreads();
    for (int c = warp; c < columns; c += BT_WARPS) {
      const int j = j0 + c, x = lane < B && j < have ? s_x[lane * line + c] : -1;
      const bool has = j < need && j != open;
      const int mine = __shfl_sync(0xffffffffu, x, max(p, 0));
      const unsigned held = __reduce_or_sync(0xffffffffu, has ? 1u << p : 0u);  // rows whose block some child has
      // (mostly a prompt's block, which all rows have: a match costs several times as much)
      const int first_x = __shfl_sync(0xffffffffu, x, 0);
      const bool alike = __all_sync(0xffffffffu, lane >= B || x == first_x) != 0;
      const unsigned same = alike ? (lane < B ? 0xffffffffu >> (32 - B) : 0u) : __match_any_sync(0xffffffffu, x), given = __ballot_sync(0xffffffffu, x >= 0 && j >= own_first);
      // (each block once, by the first of the rows that give it)
      const bool gone = ((given >> lane) & 1) != 0 && (same & held) == 0 && __ffs(same & given) - 1 == lane;
      const unsigned all = __ballot_sync(0xffffffffu, gone);
      if (lane < B) s_new[lane * line + c] = has ? mine : -1;
      if (lane == 0) s_gone[c] = all;
    }
    __syncthreads();
    for (int i = tid; i < B << shift; i += BT_THREADS) {
      const int b = i >> shift, c = i & (most - 1);
      if (c < columns) a.tables_out[static_cast<int64_t>(row0 + b) * W + j0 + c] = s_new[b * line + c];
    }
    // what is given back, by column and row
    if (warp == 0) {
      for (int c0 = 0; c0 < columns; c0 += 32) {
        const int n = c0 + lane < columns ? __popc(s_gone[c0 + lane]) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += up;
        }
        s_at[c0 + lane] = before + incl - n;
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
    __syncthreads();
    for (int c = warp; c < columns; c += BT_WARPS) {
      const unsigned all = s_gone[c];
      if ((all >> lane) & 1) a.given[static_cast<int64_t>(row0) * W + s_at[c] + __popc(all & ((1u << lane) - 1))] = s_x[lane * line + c];
    }
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
  __shared__ int s_src[BR_COPIES], s_dst[BR_COPIES], s_tokens[BR_COPIES];
  const int64_t block_bytes = bs * a.token_bytes;
  const int pieces = static_cast<int>((block_bytes + BR_PIECE - 1) / BR_PIECE);
  const int64_t per_copy = static_cast<int64_t>(a.planes) * pieces;
  for (int c0 = 0; c0 < take; c0 += BR_COPIES) {
    const int copies = min(BR_COPIES, take - c0);
    __syncthreads();  // (those before have been made)
    for (int c = tid; c < copies; c += BR_THREADS) {
      const int r = request_of(s_take, c0 + c);
      const int4 copy = a.copies[static_cast<int64_t>(r) * a.beams + c0 + c - s_take[r]];
      const int block = block_for(c0 + c);
      s_src[c] = copy.y;
      s_dst[c] = block;
      s_tokens[c] = block < 0 ? 0 : copy.w;
    }
    __syncthreads();
    const int64_t units = copies * per_copy, warps = static_cast<int64_t>(gridDim.x) * BR_WARPS;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * BR_WARPS + warp; u < units; u += warps) {
      const int c = static_cast<int>(u / per_copy), rest = static_cast<int>(u - c * per_copy), plane = rest / pieces, piece = rest - plane * pieces;
      const int64_t bytes = s_tokens[c] * a.token_bytes, from = static_cast<int64_t>(piece) * BR_PIECE;
      if (from >= bytes) continue;
      const uint4* src = reinterpret_cast<const uint4*>(a.cache + plane * a.plane_bytes + s_src[c] * block_bytes + from);
      uint4* dst = reinterpret_cast<uint4*>(a.cache + plane * a.plane_bytes + s_dst[c] * block_bytes + from);
      const int vectors = static_cast<int>(min(static_cast<int64_t>(BR_PIECE), bytes - from) / 16);
      uint4 v[BR_PIECE / 512];
#pragma unroll
      for (int e = 0; e < BR_PIECE / 512; ++e)
        if (e * 32 + lane < vectors) v[e] = src[e * 32 + lane];
#pragma unroll
      for (int e = 0; e < BR_PIECE / 512; ++e)
        if (e * 32 + lane < vectors) dst[e * 32 + lane] = v[e];
    }
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
  int chunks, warps, parts;
  int64_t maxima_bytes, bytes;
};
SelectPlan plan_select(int num_sms, int rows, int vocab, bool fp32) {
  SelectPlan p;
  // (a row may begin anywhere between two 16-byte boundaries)
  const int64_t size = fp32 ? 4 : 2;
  p.chunks = static_cast<int>((vocab * size + 16 - size + BS_CHUNK_BYTES - 1) / BS_CHUNK_BYTES);
  const int64_t total = static_cast<int64_t>(rows) * p.chunks;
  p.warps = static_cast<int>(std::min<int64_t>(total, static_cast<int64_t>(num_sms) * BS_CTAS_PER_SM * BS_WARPS));
  const int64_t least = std::max<int64_t>(1, total / std::max(1, p.warps));  // chunks of the shortest range
  p.parts = static_cast<int>(std::min<int64_t>(p.chunks, (p.chunks + least - 1) / least + 1));
  p.maxima_bytes = (total * 4 + 15) / 16 * 16;
  p.bytes = p.maxima_bytes + static_cast<int64_t>(rows) * p.parts * static_cast<int64_t>(sizeof(double2));
  return p;
}

}  // namespace

extern "C" {

int64_t b2_beam_select_workspace(b2_ctx* ctx, int n, int beams, int vocab, int picks, int fp32) {
  if (ctx == nullptr || n < 0 || beams < 1 || beams > BS_MAX_BEAMS || picks < 1 || picks > BS_MAX_PICKS || vocab < 1 || vocab > 1 << 30 || static_cast<int64_t>(n) * beams > 1 << 24) return -1;
  const int64_t chunks = static_cast<int64_t>(vocab) * (fp32 ? 4 : 2) / BS_CHUNK_BYTES + 2;
  if (chunks * n * beams >= 1ll << 31) return -1;  // (they are counted in 32 bits)
  return n == 0 ? 0 : plan_select(ctx->num_sms, n * beams, vocab, fp32 != 0).bytes;
}

int b2_beam_select(b2_ctx* ctx, const void* logits, int64_t ld, int fp32, int n, int beams, int vocab, const float* scores, const uint8_t* finished, int picks, int eos_token,
                   float* scores_out, int32_t* parents_out, int64_t* tokens_out, uint8_t* finished_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n < 0) return B2_ERR_ARG;
  if (n == 0) return B2_OK;
  const int64_t need = b2_beam_select_workspace(ctx, n, beams, vocab, picks, fp32);
  if (need < 0) return b2::set_error(B2_ERR_SHAPE, "%d requests of %d beams, %d picks of %d: at most %d beams and %d picks", n, beams, picks, vocab, BS_MAX_BEAMS, BS_MAX_PICKS);
  if (!logits || !scores || !scores_out || !parents_out || !tokens_out || !finished_out || ld < vocab) return B2_ERR_ARG;
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) return B2_ERR_ARG;
  const SelectPlan p = plan_select(ctx->num_sms, n * beams, vocab, fp32 != 0);
  char* ws = static_cast<char*>(workspace);
  const ScanArgs s{logits, ld, n * beams, beams, vocab, picks, p.chunks, p.parts, p.warps, scores, finished, reinterpret_cast<float*>(ws), reinterpret_cast<double2*>(ws + p.maxima_bytes)};
  const PickArgs k{s, eos_token, scores_out, parents_out, tokens_out, finished_out};
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  B2_CUDA(b2_launch(fp32 ? beam_scan_kernel<float> : beam_scan_kernel<__nv_bfloat16>, dim3((p.warps + BS_WARPS - 1) / BS_WARPS), dim3(BS_THREADS), 0, on, s));
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
  const bool texts = history_lens != nullptr;  // (histories without places have no address)
  if (texts ? !history_lens_out || (history_width > 0 && (!history || !history_out)) || history_stride < history_width : history || history_out || history_lens_out || tokens) return B2_ERR_ARG;
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
                      static_cast<unsigned char*>(cache), planes, plane_bytes, token_bytes, history, history_stride, texts ? history_width : 0, history_lens, tokens,
                      tables_out, lens_out, num_free_out, history_out, history_lens_out, reinterpret_cast<int2*>(ws + rows * sizeof(int4)), reinterpret_cast<int4*>(ws),
                      reinterpret_cast<int32_t*>(ws + rows * sizeof(int4) + counts_bytes)};
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  // histories: a CTA for each piece of a row, four per SM at most
  const int64_t pieces = texts ? rows * std::max(1, (history_width + BR_HISTORY - 1) / BR_HISTORY) : 0;
  const int more = static_cast<int>(std::min<int64_t>(pieces, 4 * ctx->num_sms));
  if (n + more > 0) B2_CUDA(b2_launch(beam_tables_kernel, dim3(n + more), dim3(BT_THREADS), 0, on, a));
  const int64_t most = rows * planes * ((block_size * token_bytes + BR_PIECE - 1) / BR_PIECE) / (BR_THREADS / 32);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4 * ctx->num_sms, most)));
  B2_CUDA(b2_launch(beam_move_kernel, dim3(grid), dim3(BR_THREADS), 2 * (n + 1) * sizeof(int), on, a));
  return B2_OK;
}

}  // extern "C"
