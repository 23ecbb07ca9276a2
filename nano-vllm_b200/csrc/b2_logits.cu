// Rules on logits between the LM head and the sampler: penalties for repeated tokens, biases, grammar masks.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// For a row of logits that belongs to request s, token v, with `count` its occurrences in the request's output (and on the row's path of
// drafted tokens) and `seen` whether it occurs there or in the prompt, in 32 bits and in this order:
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * count;   x = count > 0 ? x - presence : x
//   x = x + bias(v)                   the last entry of v in the request's list
//   x = allowed ? x : -inf
// and one rounding to the logits' type.  Logits that no rule touches are copied bit for bit.
//
// Bound: HBM, logits in and out once.  Two kernels:
//
// mask_logits_kernel moves all logits, 16-byte vectors with the forbidden tokens masked a word at a time.  It is left out where out is the
// logits and there is no mask.
//
// rules_kernel stores the few that history, biases and paths touch, over what the first one stored.  A CTA takes every P-th token of
// one request: it counts the history into a word of shared memory for each of its tokens (all of it is read, its own tokens count; text repeats low
// ids, and they are spread over the P CTAs), and whoever finds a word at zero lists its token.  The list is worked through a token to a thread, for four
// of the request's rows - a tree's nodes - at a time.  A token on a row's path of drafted tokens is marked: it is not the list's, but the thread's of the
// path's first node that has it.  All that needs no logits stored is done while the first kernel is still at work.  No counts live in memory between calls:
// the state of a request is the list of its tokens.  Counting works on whole numbers and every store is one thread's, so that the order changes nothing.
//
// (One kernel, a CTA for a slice of the vocabulary that counts, changes the touched logits in shared memory and masks them on their way out: 23 us for
// 64 rows of 151936 with all rules, 91 for 512 rows of trees.  Its loads were in flight for a fraction of its time.)
// ---------------------------------------------------------------------------
constexpr int ML_THREADS = 256, ML_CTAS_PER_SM = 4, ML_UNROLL = 4;
constexpr int RL_THREADS = 512, RL_TOKENS = 16384;  // of one CTA, at most
constexpr int RL_ROWS = 4;
// a token's word: how often it occurs in the output, the last place of its id in the request's list of biases (from 1), whether the prompt has it
constexpr int AL_COUNT_BITS = 19, AL_BIAS_BITS = 12;
constexpr uint32_t AL_COUNT = (1u << AL_COUNT_BITS) - 1, AL_PROMPT = 0x80000000u;
static_assert(AL_COUNT_BITS + AL_BIAS_BITS == 31, "a word");

struct LogitArgs {
  const void* logits;
  void* out;
  int64_t ld, ld_out;
  int rows, vocab, n_seqs;
  const int32_t* cu;  // null: row i is request i
  const int64_t* history;
  int64_t history_stride;
  int history_width;
  const int32_t *history_lens, *prompt_lens;
  const float *repetition, *presence, *frequency;
  const int64_t* bias_ids;
  int64_t bias_stride;
  int n_bias;
  const float* bias_values;
  int64_t bias_value_stride;
  const int32_t* allowed;
  int64_t allowed_stride;
  const int64_t *drafts, *tree_mask;
  int64_t mask_stride;
  int words;
  // rules_kernel: 2^part_bits CTAs share a request's tokens, as many times `splits` for parts of its rows; after the first kernel
  int part_bits, splits, second;
};

template <class T>
struct Logit;
template <>
struct Logit<uint16_t> {
  static constexpr uint32_t kMinusInf = 0xff80ff80u;  // as many as a word holds
  static __device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
  // ones in the halves whose bit is set: the bits as the signs of two bytes, which a permutation spreads
  static __device__ __forceinline__ uint32_t keep(uint32_t bits) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(r) : "r"((bits & 3) * 0x4080u));
    return r;
  }
};
template <>
struct Logit<uint32_t> {
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static __device__ __forceinline__ float widen(uint32_t x) { return __uint_as_float(x); }
  static __device__ __forceinline__ uint32_t narrow(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ uint32_t keep(uint32_t bits) { return 0u - (bits & 1); }
};

template <class T>
__global__ void __launch_bounds__(ML_THREADS, ML_CTAS_PER_SM) mask_logits_kernel(const LogitArgs a) {
  constexpr int V = 16 / sizeof(T), CHUNK = 32 * V, PAIR = 4 / sizeof(T);
  b2::pdl_wait();
  b2::pdl_launch_dependents();  // (only now: the next kernel reads the inputs ahead of its own wait)
  const int lane = threadIdx.x & 31, warps = gridDim.x * (ML_THREADS / 32);
  const int ruled = a.cu != nullptr ? __ldg(a.cu + a.n_seqs) : a.rows;  // rows behind the last request are copied
  const int chunks = (a.vocab + CHUNK - 1) / CHUNK, per_row = (chunks + ML_UNROLL - 1) / ML_UNROLL;
  // a warp takes ML_UNROLL chunks of a row at a time: 32 vectors where the chunk is whole and both rows have their 16-byte boundaries in common,
  // but for the elements before the first boundary and behind the last, which go one by one, as all do otherwise
  int64_t unit = blockIdx.x * (ML_THREADS / 32) + (threadIdx.x >> 5);
  int row = static_cast<int>(unit / per_row), at = static_cast<int>(unit - static_cast<int64_t>(row) * per_row);
  const int step_rows = warps / per_row, step_at = warps - step_rows * per_row;
  while (row < a.rows) {
    const T* const in = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld;
    T* const out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.ld_out;
    const uint8_t* const bits = reinterpret_cast<const uint8_t*>(a.allowed + static_cast<int64_t>(row) * a.allowed_stride);
    const bool masked = a.allowed != nullptr && row < ruled;
    const bool same = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / static_cast<int>(sizeof(T));
    auto element = [&](int t) { out[t] = !masked || ((__ldg(bits + (t >> 3)) >> (t & 7)) & 1) ? in[t] : static_cast<T>(Logit<T>::kMinusInf); };
    auto word = [&](uint32_t w, uint32_t b) {
      const uint32_t keep = Logit<T>::keep(b);
      return (w & keep) | (Logit<T>::kMinusInf & ~keep);
    };
    const int t0 = at * ML_UNROLL * CHUNK;
    if (same && t0 + ML_UNROLL * CHUNK <= a.vocab) {
      uint4 x[ML_UNROLL];
      uint32_t yes[ML_UNROLL];
      const bool vector = head == 0 || lane < 31;
#pragma unroll
      for (int i = 0; i < ML_UNROLL; ++i) {
        const int t = t0 + i * CHUNK + head + lane * V;
        if (vector) {
          x[i] = *reinterpret_cast<const uint4*>(in + t);
          if (masked) {
            yes[i] = __ldg(bits + (t >> 3)) >> (t & 7);
            if ((t & 7) + V > 8) yes[i] |= static_cast<uint32_t>(__ldg(bits + (t >> 3) + 1)) << (8 - (t & 7));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ML_UNROLL; ++i) {
        const int t = t0 + i * CHUNK;
        if (masked) x[i] = make_uint4(word(x[i].x, yes[i]), word(x[i].y, yes[i] >> PAIR), word(x[i].z, yes[i] >> 2 * PAIR), word(x[i].w, yes[i] >> 3 * PAIR));
        if (vector) *reinterpret_cast<uint4*>(out + t + head + lane * V) = x[i];
        if (head > 0 && lane < V) element(lane < head ? t + lane : t + CHUNK - V + lane);
      }
    } else {
#pragma unroll 4
      for (int t = t0 + lane; t < min(t0 + ML_UNROLL * CHUNK, a.vocab); t += 32) element(t);
    }
    row += step_rows;
    at += step_at;
    if (at >= per_row) {
      at -= per_row;
      ++row;
    }
  }
}

// shared memory: words of the tokens, the marks of RL_ROWS rows, the list
__host__ __device__ constexpr int rules_tokens(int vocab, int part_bits) { return ((vocab - 1) >> part_bits) + 1; }
constexpr size_t rules_smem(int tokens) { return static_cast<size_t>((tokens + 3) / 4 * 4) * 4 + static_cast<size_t>(RL_ROWS) * ((tokens + 31) / 32) * 4 + static_cast<size_t>(tokens) * 2; }

template <class T>
__global__ void __launch_bounds__(RL_THREADS) rules_kernel(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t s_words[];
  __shared__ int s_listed;
  const int tokens = rules_tokens(a.vocab, a.part_bits), padded = (tokens + 3) / 4 * 4, mark_words = (tokens + 31) / 32;
  uint32_t* const s_marks = s_words + padded;
  uint16_t* const s_list = reinterpret_cast<uint16_t*>(s_marks + RL_ROWS * mark_words);
  const int tid = threadIdx.x;
  const uint32_t part = blockIdx.x & ((1u << a.part_bits) - 1);
  const int s = static_cast<int>((blockIdx.x >> a.part_bits) / a.splits), split = static_cast<int>((blockIdx.x >> a.part_bits) - s * a.splits);
  b2::pdl_launch_dependents();
  if (!a.second) b2::pdl_wait();

  for (int i = tid; i < padded / 4; i += RL_THREADS) reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < RL_ROWS * mark_words; i += RL_THREADS) s_marks[i] = 0;
  if (tid == 0) s_listed = 0;
  // the request's rows, and this CTA's
  const int node0 = a.cu != nullptr ? max(0, __ldg(a.cu + s)) : s, end = a.cu != nullptr ? min(a.rows, __ldg(a.cu + s + 1)) : s + 1;
  const int per = (max(0, end - node0) + a.splits - 1) / a.splits, row0 = node0 + split * per, row1 = min(end, row0 + per);
  const int nodes = a.drafts != nullptr ? min(end - node0, 64 * a.words) : 0;
  if (row0 >= row1) {
    if (a.second) b2::pdl_wait();  // (this kernel must not be over before the first one is: what follows waits for this one)
    return;
  }
  // a token's place among this CTA's, or -1, and back
  auto place_of = [&](int lo, int hi) {
    return hi == 0 && static_cast<uint32_t>(lo) < static_cast<uint32_t>(a.vocab) && (lo & ((1u << a.part_bits) - 1)) == part ? lo >> a.part_bits : -1;
  };
  auto token_at = [&](int e) { return (e << a.part_bits) + static_cast<int>(part); };
  auto id = [&](const int64_t* ids, int64_t i) {
    const int2 t = __ldg(reinterpret_cast<const int2*>(ids) + i);
    return place_of(t.x, t.y);
  };
  // adds a token to the list whose word was zero
  auto list = [&](uint32_t before, int e) {
    if (before == 0) s_list[atomicAdd(&s_listed, 1)] = static_cast<uint16_t>(e);
  };
  const int64_t* const text = a.history + static_cast<int64_t>(s) * a.history_stride;
  const int n = a.history != nullptr ? max(0, min(__ldg(a.history_lens + s), a.history_width)) : 0, prompt = a.prompt_lens != nullptr ? __ldg(a.prompt_lens + s) : 0;
  const float repetition = a.repetition != nullptr ? __ldg(a.repetition + s) : 1.f, presence = a.presence != nullptr ? __ldg(a.presence + s) : 0.f,
              frequency = a.frequency != nullptr ? __ldg(a.frequency + s) : 0.f;
  __syncthreads();
  if (a.n_bias > 0) {
    for (int i = tid; i < a.n_bias; i += RL_THREADS) {
      const int e = id(a.bias_ids, s * a.bias_stride + i);
      if (e >= 0) list(atomicMax(s_words + e, static_cast<uint32_t>(i + 1) << AL_COUNT_BITS), e);
    }
    __syncthreads();  // (places first: counts and prompt bits are added to words that hold them)
  }
  auto count = [&](int e, int i) {
    if (e >= 0) list(i < prompt ? atomicOr(s_words + e, AL_PROMPT) : atomicAdd(s_words + e, 1u), e);
  };
  // two tokens a load, eight loads on their way at once; the first where it is not on a 16-byte boundary, and an odd last one
  const int skip = n > 0 && (reinterpret_cast<uintptr_t>(text) & 15) != 0 ? 1 : 0, pairs = (n - skip) >> 1;
  const int4* const two = reinterpret_cast<const int4*>(text + skip);
  for (int p0 = tid; p0 < pairs; p0 += 8 * RL_THREADS) {
    int4 t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = p0 + k * RL_THREADS < pairs ? __ldg(two + p0 + k * RL_THREADS) : make_int4(-1, -1, -1, -1);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = skip + 2 * (p0 + k * RL_THREADS);
      count(place_of(t[k].x, t[k].y), i);
      count(place_of(t[k].z, t[k].w), i + 1);
    }
  }
  if (skip && tid == 0) count(id(text, 0), 0);
  if (((n - skip) & 1) && tid == 32) count(id(text, n - 1), n - 1);
  __syncthreads();
  const int listed = s_listed;
  if (a.second) b2::pdl_wait();

  // Where out is the logits, a logit that is read here is what it was, or masked, as it then is in the end.
  auto in_row = [&](int row) { return static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld; };
  auto out_row = [&](int row) { return static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.ld_out; };
  auto permitted = [&](int row, int t) { return a.allowed == nullptr || ((__ldg(a.allowed + static_cast<int64_t>(row) * a.allowed_stride + (t >> 5)) >> (t & 31)) & 1); };
  auto bias_of = [&](uint32_t w) {
    const uint32_t place = (w & ~AL_PROMPT) >> AL_COUNT_BITS;
    return place != 0 ? __ldg(a.bias_values + s * a.bias_value_stride + place - 1) : 0.f;
  };
  auto value = [&](T raw, bool yes, uint32_t w, uint32_t more, float bias) {
    const uint32_t count = (w & AL_COUNT) + more;
    float y = Logit<T>::widen(raw);
    if ((count != 0 || (w & AL_PROMPT)) && a.repetition != nullptr) y = y > 0.f ? __fdiv_rn(y, repetition) : y * repetition;
    if (count != 0) {
      y = __fsub_rn(y, __fmul_rn(frequency, static_cast<float>(count)));
      y = __fsub_rn(y, presence);
    }
    if ((w & ~AL_PROMPT) >> AL_COUNT_BITS) y += bias;
    return yes ? Logit<T>::narrow(y) : static_cast<T>(Logit<T>::kMinusInf);
  };
  auto path = [&](int row) { return reinterpret_cast<const unsigned long long*>(a.tree_mask + static_cast<int64_t>(row) * a.mask_stride); };
  auto on_path = [&](int row, int k) { return (__ldg(path(row) + (k >> 6)) >> (k & 63)) & 1 ? id(a.drafts, node0 + k) : -1; };
  for (int r0 = row0; r0 < row1; r0 += RL_ROWS) {
    const int here = min(RL_ROWS, row1 - r0);
    if (nodes > 0) {
      for (int i = tid; i < here * nodes; i += RL_THREADS) {
        const int e = on_path(r0 + i / nodes, i % nodes);
        if (e >= 0) atomicOr(s_marks + i / nodes * mark_words + (e >> 5), 1u << (e & 31));
      }
      __syncthreads();
    }
    for (int i = tid; i < listed; i += RL_THREADS) {
      const int e = s_list[i], t = token_at(e);
      const uint32_t w = s_words[e];
      T raw[RL_ROWS];
      bool yes[RL_ROWS];
#pragma unroll
      for (int r = 0; r < RL_ROWS; ++r)
        if (r < here) {
          raw[r] = in_row(r0 + r)[t];
          yes[r] = permitted(r0 + r, t);
        }
      const float bias = bias_of(w);
#pragma unroll
      for (int r = 0; r < RL_ROWS; ++r)
        if (r < here && !((s_marks[r * mark_words + (e >> 5)] >> (e & 31)) & 1)) out_row(r0 + r)[t] = value(raw[r], yes[r], w, 0, bias);
    }
    if (nodes > 0) {
      for (int i = tid; i < here * nodes; i += RL_THREADS) {
        const int row = r0 + i / nodes, k = i % nodes, e = on_path(row, k);
        if (e < 0) continue;
        uint32_t times = 0;
        bool first = true;
        for (int j0 = 0; j0 < nodes; j0 += 64)
          for (uint64_t bits = __ldg(path(row) + (j0 >> 6)); bits != 0; bits &= bits - 1) {
            const int j = j0 + __ffsll(bits) - 1;
            if (j >= nodes) break;
            if (id(a.drafts, node0 + j) != e) continue;
            ++times;
            first = first && j >= k;
          }
        if (!first) continue;
        const int t = token_at(e);
        const uint32_t w = s_words[e];
        out_row(row)[t] = value(in_row(row)[t], permitted(row, t), w, times, bias_of(w));
      }
      if (r0 + RL_ROWS < row1) {
        __syncthreads();
        for (int i = tid; i < RL_ROWS * mark_words; i += RL_THREADS) s_marks[i] = 0;
        __syncthreads();
      }
    }
  }
}

// sms: the device's
int configure_once(int* sms) {
  static std::atomic<int> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  *sms = done[dev].load(std::memory_order_acquire);
  if (*sms == 0) {
    B2_CUDA(cudaFuncSetAttribute(rules_kernel<uint16_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, rules_smem(RL_TOKENS)));
    B2_CUDA(cudaFuncSetAttribute(rules_kernel<uint32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, rules_smem(RL_TOKENS)));
    B2_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    done[dev].store(*sms, std::memory_order_release);
  }
  return B2_OK;
}

}  // namespace

extern "C" int b2_adjust_logits(const void* logits, int64_t ld, void* out, int64_t ld_out, int fp32, int rows, int vocab, const b2_logit_rules* r, void* stream) {
  if (rows < 0 || vocab < 0 || ld < vocab || ld_out < vocab || r == nullptr) return B2_ERR_ARG;
  if (rows == 0 || vocab == 0) return B2_OK;
  if (!logits || !out || r->n_seqs < 0 || (r->cu_seqlens == nullptr && r->n_seqs != rows)) return B2_ERR_ARG;
  const uintptr_t align = fp32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & align) return B2_ERR_ARG;
  if (r->history != nullptr && (r->history_width < 0 || r->history_lens == nullptr)) return B2_ERR_ARG;
  if (r->n_bias < 0 || (r->n_bias > 0 && (!r->bias_ids || !r->bias_values))) return B2_ERR_ARG;
  if (r->allowed_mask != nullptr && r->allowed_stride < (vocab + 31) / 32) return B2_ERR_ARG;
  if (r->draft_tokens != nullptr && (!r->tree_mask || !r->cu_seqlens || r->mask_words <= 0 || r->mask_stride < r->mask_words || r->mask_words > 1 << 12)) return B2_ERR_ARG;
  if (r->n_bias >= 1 << AL_BIAS_BITS || (r->history != nullptr ? r->history_width : 0) + 64ll * (r->draft_tokens != nullptr ? r->mask_words : 0) > AL_COUNT)
    return b2::set_error(B2_ERR_SHAPE, "at most %d biases, and %d tokens of history and path", (1 << AL_BIAS_BITS) - 1, AL_COUNT);
  int sms = 0;
  const int rc = configure_once(&sms);
  if (rc != B2_OK) return rc;
  LogitArgs a{};
  a.logits = logits;
  a.out = out;
  a.ld = ld;
  a.ld_out = ld_out;
  a.rows = rows;
  a.vocab = vocab;
  a.n_seqs = r->n_seqs;
  a.cu = r->cu_seqlens;
  a.history = r->history;
  a.history_stride = r->history_stride;
  a.history_width = r->history_width;
  a.history_lens = r->history_lens;
  a.prompt_lens = r->prompt_lens;
  a.repetition = r->repetition_penalty;
  a.presence = r->presence_penalty;
  a.frequency = r->frequency_penalty;
  a.bias_ids = r->bias_ids;
  a.bias_stride = r->bias_stride;
  a.n_bias = r->n_bias;
  a.bias_values = r->bias_values;
  a.bias_value_stride = r->bias_value_stride;
  a.allowed = r->allowed_mask;
  a.allowed_stride = r->allowed_stride;
  a.drafts = r->draft_tokens;
  a.tree_mask = r->tree_mask;
  a.mask_stride = r->mask_stride;
  a.words = r->mask_words;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (logits != out || a.allowed != nullptr) {
    const int64_t chunks = (static_cast<int64_t>(vocab) + (fp32 ? 128 : 256) * ML_UNROLL - 1) / ((fp32 ? 128 : 256) * ML_UNROLL);
    const int64_t blocks = (chunks * rows + ML_THREADS / 32 - 1) / (ML_THREADS / 32);
    const auto kernel = fp32 ? mask_logits_kernel<uint32_t> : mask_logits_kernel<uint16_t>;
    B2_CUDA(b2_launch(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, static_cast<int64_t>(sms) * ML_CTAS_PER_SM))), dim3(ML_THREADS), 0, on, a));
    a.second = 1;
  }
  if ((a.history != nullptr || a.n_bias > 0 || a.drafts != nullptr) && a.n_seqs > 0) {
    while (rules_tokens(vocab, a.part_bits) > RL_TOKENS) ++a.part_bits;
    // a request's rows in so many parts that there are two CTAs for every SM, but no fewer than RL_ROWS of them to a CTA
    const int64_t items = static_cast<int64_t>(a.n_seqs) << a.part_bits;
    a.splits = a.cu == nullptr ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((2 * sms + items - 1) / items, (rows / a.n_seqs + RL_ROWS - 1) / RL_ROWS)));
    if (items * a.splits >= 1ll << 31) return b2::set_error(B2_ERR_SHAPE, "%d requests over %d tokens", a.n_seqs, vocab);
    const auto kernel = fp32 ? rules_kernel<uint32_t> : rules_kernel<uint16_t>;
    B2_CUDA(b2_launch(kernel, dim3(static_cast<unsigned>(items * a.splits)), dim3(RL_THREADS), rules_smem(rules_tokens(vocab, a.part_bits)), on, a));
  }
  return B2_OK;
}
