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
// Bound: HBM, logits in and out once.  A step is a row's piece of a slice of the vocabulary, 16 KB; a CTA takes an even range of the steps, slice
// after slice.  The piece of the next step is on its way to registers while a step runs:
//   the request's history is counted into a word of shared memory for each token of the slice (all of it is read, the tokens of the slice
//   count), and whoever finds a word at zero lists its token; rows of one request - a tree's nodes - follow each other and share the counts and the
//   list, with the tokens of their paths added and taken out again
//   the piece lies in shared memory while the listed tokens get their new values, a thread each
//   and leaves in 16-byte vectors, with the forbidden tokens masked a word at a time
// No counts live in memory between calls: the state of a request is the list of its tokens.  Counting works on whole numbers and every listed
// token is one thread's, so that the order changes nothing.
//
// Measured (one row of 151936 with penalties and biases / 33 rows of 50257 in fp32 after 15000 to 30000 tokens / 64 rows with all rules / 512 rows of 32 trees):
// device time of calls one after the other 3.9 / 29 / 22 / 86 us; the bytes alone take - / 3 / 6.4 / 49.  What is left for long histories is the counting: each
// of 13 or 19 slices reads all of them, and no unit is full (issue slots 55 and 49 %, HBM 5 and 11 %); for the trees the barriers between a step's phases, where
// a warp waits longest (4.7 of 13.7 cycles an instruction).  Tried, passes timed with the host, on which this kernel took 7.0 / 30 / 22 / 87: a CTA for
// each step, loads and phases one after the other 7 / 26 / 33 / 220 (better for the 33 rows, which have no drafts and few rules, and for nothing else); 512 threads,
// whose registers spill, 172 for the trees; pieces by bulk copies through a ring 7 / 34 / 26 / 88; one kernel that copies and masks and one that counts and
// stores the listed tokens 11 / 26 / 20 / 116; lists from a kernel of their own 12 / 32 / 26 / 79.
// ---------------------------------------------------------------------------
constexpr int AL_THREADS = 256;
constexpr int AL_PIECE = 16384;  // bytes
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
  int words, slices;
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

// n <= 8 bits of a bitmap from bit i on
__device__ __forceinline__ uint32_t bits_at(const uint32_t* map, int i, int n) {
  return __funnelshift_r(map[i >> 5], map[(i >> 5) + 1], i & 31) & ((1u << n) - 1);
}

template <class T>
struct Slice {
  static constexpr int TOKENS = AL_PIECE / sizeof(T);
  static constexpr size_t SMEM = TOKENS * (sizeof(uint32_t) + sizeof(uint16_t)) + AL_PIECE + 16;
  static constexpr int CTAS_PER_SM = 3;  // (64 and 40 KB of shared memory; with 64 registers instead of 85 the threads would spill, which costs more)
};

template <class T>
__global__ void __launch_bounds__(AL_THREADS, Slice<T>::CTAS_PER_SM) adjust_logits_kernel(const LogitArgs a) {
  constexpr int TOKENS = Slice<T>::TOKENS, V = 16 / sizeof(T), PER = AL_PIECE / 16 / AL_THREADS, PAIR = 4 / sizeof(T);
  extern __shared__ __align__(16) uint32_t s_words[];  // [TOKENS] words of the tokens, the list of the touched ones, the row's logits
  uint16_t* const s_list = reinterpret_cast<uint16_t*>(s_words + TOKENS);
  T* const s_logits = reinterpret_cast<T*>(s_list + TOKENS);
  __shared__ uint32_t s_allowed[TOKENS / 32 + 1];
  __shared__ int s_listed[2];  // entries of the list: of the request's history and biases, and with the row's path
  static_assert(AL_THREADS >= TOKENS / 32, "a word of the mask to a thread");
  const int tid = threadIdx.x;
  const bool counts = a.history != nullptr || a.n_bias > 0 || a.drafts != nullptr;
  if (counts) {
    for (int i = tid; i < TOKENS / 4; i += AL_THREADS) reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) s_listed[0] = s_listed[1] = 0;
  }
  b2::pdl_launch_dependents();
  b2::pdl_wait();

  // this CTA's steps: slice after slice, the rows of each in order
  const int64_t steps = static_cast<int64_t>(a.rows) * a.slices, first = steps * blockIdx.x / gridDim.x;
  int todo = static_cast<int>(steps * (blockIdx.x + 1) / gridDim.x - first);
  int slice = static_cast<int>(first / a.rows), row = static_cast<int>(first - static_cast<int64_t>(slice) * a.rows);
  struct Piece {
    const T* in;
    T* out;
    int len, head, vectors;  // 16-byte vectors where both rows allow them, the elements before (head) and behind one by one
  };
  auto piece = [&](int slice, int row) {
    Piece p;
    p.in = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld + slice * TOKENS;
    p.out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.ld_out + slice * TOKENS;
    p.len = min(TOKENS, a.vocab - slice * TOKENS);
    const bool same = ((reinterpret_cast<uintptr_t>(p.in) ^ reinterpret_cast<uintptr_t>(p.out)) & 15) == 0;
    p.head = same ? min(p.len, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p.in) & 15)) & 15) / static_cast<int>(sizeof(T))) : p.len;
    p.vectors = (p.len - p.head) / V;
    return p;
  };
  uint4 x[PER];
  uint32_t allowed = 0u;
  auto fetch = [&](const Piece& p, int slice, int row) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * AL_THREADS + tid < p.vectors) x[i] = *reinterpret_cast<const uint4*>(p.in + p.head + (i * AL_THREADS + tid) * V);
    if (a.allowed != nullptr)
      allowed = tid < (p.len + 31) / 32 ? __ldg(a.allowed + static_cast<int64_t>(row) * a.allowed_stride + slice * (TOKENS / 32) + tid) : 0u;
  };
  // adds a token to the list whose word was zero
  auto list = [&](uint32_t before, int e) {
    if (before == 0) s_list[atomicAdd(s_listed + 1, 1)] = static_cast<uint16_t>(e);
  };
  int seq = -1, seq_end = 0, node0 = 0, nodes = 0;  // the request whose tokens the words hold, the row behind its last
  int my_draft = -1;                                // this thread's node's token: its place in the slice
  uint64_t my_path = 0;                             // the word of the row's mask that has this thread's node
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  Piece now = piece(slice, row);
  fetch(now, slice, row);
  for (; todo > 0; --todo) {
    const int v0 = slice * TOKENS, len = now.len;
    // a token's place in the slice, or -1
    auto place_of = [&](int lo, int hi) {
      const uint32_t e = static_cast<uint32_t>(lo) - static_cast<uint32_t>(v0);
      return hi == 0 && e < static_cast<uint32_t>(len) ? static_cast<int>(e) : -1;
    };
    auto id = [&](const int64_t* ids, int64_t i) {
      const int2 t = __ldg(reinterpret_cast<const int2*>(ids) + i);
      return place_of(t.x, t.y);
    };
    auto path_word = [&](int r, int k) { return __ldg(reinterpret_cast<const unsigned long long*>(a.tree_mask + static_cast<int64_t>(r) * a.mask_stride) + (k >> 6)); };

    // ---- the row's request ----
    int s = row;
    bool ruled = true;  // rows before the first request and behind the last are copied
    if (a.cu != nullptr) {
      if (seq >= 0 && row >= node0 && row < seq_end) {
        s = seq;
      } else {
        s = 0;
        int hi = a.n_seqs;  // the first request whose rows end behind this one
        while (s < hi) {
          const int mid = (s + hi) >> 1;
          if (__ldg(a.cu + mid + 1) > row) hi = mid;
          else s = mid + 1;
        }
        ruled = s < a.n_seqs && __ldg(a.cu + s) <= row;
      }
    }
    if (ruled && s != seq) {
      seq = s;
      seq_end = row + 1;
      const int64_t* const text = a.history + static_cast<int64_t>(s) * a.history_stride;
      const int n = a.history != nullptr ? max(0, min(__ldg(a.history_lens + s), a.history_width)) : 0, prompt = a.prompt_lens != nullptr ? __ldg(a.prompt_lens + s) : 0;
      // two tokens a load, two loads on their way at once; the first token where it is not on a 16-byte boundary, and an odd last one
      const int skip = n > 0 && (reinterpret_cast<uintptr_t>(text) & 15) != 0 ? 1 : 0, pairs = (n - skip) >> 1;
      int4 two[2];
      auto load = [&](int p0) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          two[k] = p0 + k * AL_THREADS < pairs ? __ldg(reinterpret_cast<const int4*>(text + skip) + p0 + k * AL_THREADS) : make_int4(-1, -1, -1, -1);
      };
      load(tid);
      repetition = a.repetition != nullptr ? __ldg(a.repetition + s) : 1.f;
      presence = a.presence != nullptr ? __ldg(a.presence + s) : 0.f;
      frequency = a.frequency != nullptr ? __ldg(a.frequency + s) : 0.f;
      if (a.cu != nullptr) {
        node0 = max(0, __ldg(a.cu + s));
        seq_end = min(a.rows, __ldg(a.cu + s + 1));
        nodes = a.drafts != nullptr ? min(seq_end - node0, 64 * a.words) : 0;
        my_draft = tid < nodes ? id(a.drafts, node0 + tid) : -1;
        if (my_draft >= 0) my_path = path_word(row, tid);
      }
      __syncthreads();  // (the words are zero)
      if (a.n_bias > 0) {
        for (int i = tid; i < a.n_bias; i += AL_THREADS) {
          const int e = id(a.bias_ids, s * a.bias_stride + i);
          if (e >= 0) list(atomicMax(s_words + e, static_cast<uint32_t>(i + 1) << AL_COUNT_BITS), e);
        }
        __syncthreads();  // (places first: counts and prompt bits are added to words that hold them)
      }
      auto count = [&](int e, int i) { return e < 0 ? 1u : i < prompt ? atomicOr(s_words + e, AL_PROMPT) : atomicAdd(s_words + e, 1u); };
      for (int p0 = tid; p0 < pairs; p0 += 2 * AL_THREADS) {
        int e[4];
        uint32_t before[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          e[2 * k] = place_of(two[k].x, two[k].y);
          e[2 * k + 1] = place_of(two[k].z, two[k].w);
        }
        load(p0 + 2 * AL_THREADS);
#pragma unroll
        for (int k = 0; k < 4; ++k) before[k] = count(e[k], skip + 2 * (p0 + (k >> 1) * AL_THREADS) + (k & 1));  // (four on their way before the first is asked for)
#pragma unroll
        for (int k = 0; k < 4; ++k) list(before[k], e[k]);
      }
      auto one = [&](int i) {
        const int e = id(text, i);
        list(count(e, i), e);
      };
      if (skip && tid == 0) one(0);
      if (((n - skip) & 1) && tid == 32) one(n - 1);
      if (a.cu != nullptr) {  // (for its other rows)
        __syncthreads();
        if (tid == 0) s_listed[0] = s_listed[1];
        __syncthreads();
      }
    }
    // ---- the drafted tokens that this row's node sees, as output; afterwards they are taken out again ----
    const bool drafted = ruled && nodes > 0, masked = ruled && a.allowed != nullptr;
    auto on_path = [&](int k, int& e) {
      e = k == tid ? my_draft : id(a.drafts, node0 + k);
      return e >= 0 && (((k == tid ? my_path : path_word(row, k)) >> (k & 63)) & 1);
    };
    if (drafted)
      for (int k = tid, e; k < nodes; k += AL_THREADS)
        if (on_path(k, e)) list(atomicAdd(s_words + e, 1u), e);

    // ---- the piece in shared memory, and the next one on its way ----
    const int head = now.head, vectors = now.vectors, tail = head + vectors * V;
    T* const stage = s_logits + (V - head % V) % V;  // element `head` on a 16-byte boundary
    const T* const in = now.in;
    T* const out = now.out;
    if (masked && tid < TOKENS / 32) s_allowed[tid] = allowed;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * AL_THREADS + tid < vectors) *reinterpret_cast<uint4*>(stage + head + (i * AL_THREADS + tid) * V) = x[i];
    for (int e = tid; e < head; e += AL_THREADS) stage[e] = in[e];
    for (int e = tail + tid; e < len; e += AL_THREADS) stage[e] = in[e];
    const bool more = todo > 1, turn = row + 1 == a.rows;
    const int next_slice = turn ? slice + 1 : slice, next_row = turn ? 0 : row + 1;
    if (more) {
      now = piece(next_slice, next_row);
      fetch(now, next_slice, next_row);
    }
    __syncthreads();

    // ---- the listed tokens ----
    if (ruled && counts) {
      // the words are made zero for the next request where this one has no row to come
      const bool clear = !(more && !turn && next_row < seq_end);
      const int listed = s_listed[1];
      for (int i = tid; i < listed; i += AL_THREADS) {
        const int e = s_list[i];
        const uint32_t w = s_words[e], count = w & AL_COUNT, place = (w & ~AL_PROMPT) >> AL_COUNT_BITS;
        if (clear) s_words[e] = 0;
        const float bias = place != 0 ? __ldg(a.bias_values + s * a.bias_value_stride + place - 1) : 0.f;
        float y = Logit<T>::widen(stage[e]);
        if ((count != 0 || (w & AL_PROMPT)) && a.repetition != nullptr) y = y > 0.f ? __fdiv_rn(y, repetition) : y * repetition;
        if (count != 0) {
          y = __fsub_rn(y, __fmul_rn(frequency, static_cast<float>(count)));
          y = __fsub_rn(y, presence);
        }
        if (place != 0) y += bias;
        stage[e] = Logit<T>::narrow(y);
      }
      if (clear) seq = -1;
      __syncthreads();
      if (drafted && !clear) {
        for (int k = tid, e; k < nodes; k += AL_THREADS)
          if (on_path(k, e)) atomicSub(s_words + e, 1u);
        if (my_draft >= 0) my_path = path_word(next_row, tid);
      }
      if (tid == 0) s_listed[1] = clear ? 0 : s_listed[0];
    }

    // ---- out ----
    auto word = [&](uint32_t w, uint32_t bits) {
      const uint32_t keep = Logit<T>::keep(bits);
      return (w & keep) | (Logit<T>::kMinusInf & ~keep);
    };
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = i * AL_THREADS + tid;
      if (k >= vectors) break;
      uint4 w = *reinterpret_cast<const uint4*>(stage + head + k * V);
      if (masked) {
        const uint32_t bits = bits_at(s_allowed, head + k * V, V);
        w = make_uint4(word(w.x, bits), word(w.y, bits >> PAIR), word(w.z, bits >> 2 * PAIR), word(w.w, bits >> 3 * PAIR));
      }
      *reinterpret_cast<uint4*>(out + head + k * V) = w;
    }
    auto element = [&](int e) { out[e] = !masked || ((s_allowed[e >> 5] >> (e & 31)) & 1) ? stage[e] : static_cast<T>(Logit<T>::kMinusInf); };
    for (int e = tid; e < head; e += AL_THREADS) element(e);
    for (int e = tail + tid; e < len; e += AL_THREADS) element(e);
    slice = next_slice;
    row = next_row;
    __syncthreads();  // (the next row's logits take their place)
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
    B2_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<uint16_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, Slice<uint16_t>::SMEM));
    B2_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<uint32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, Slice<uint32_t>::SMEM));
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
  const int tokens = fp32 ? Slice<uint32_t>::TOKENS : Slice<uint16_t>::TOKENS;
  a.slices = (vocab + tokens - 1) / tokens;
  const int64_t ctas = static_cast<int64_t>(sms) * (fp32 ? Slice<uint32_t>::CTAS_PER_SM : Slice<uint16_t>::CTAS_PER_SM);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(static_cast<int64_t>(rows) * a.slices, ctas)));
  B2_CUDA(b2_launch(fp32 ? adjust_logits_kernel<uint32_t> : adjust_logits_kernel<uint16_t>, grid, dim3(AL_THREADS), fp32 ? Slice<uint32_t>::SMEM : Slice<uint16_t>::SMEM, on, a));
  return B2_OK;
}
