// Rules on logits between the LM head and the sampler: penalties for repeated tokens, biases, grammar masks.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace {

// ---------------------------------------------------------------------------
// adjust_logits_kernel
//
// For a row of logits that belongs to request s, token v, with `count` its occurrences in the request's output (and on the row's path of
// drafted tokens) and `seen` whether it occurs there or in the prompt, in 32 bits and in this order:
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * count;   x = count > 0 ? x - presence : x
//   x = x + bias(v)                   the last entry of v in the request's list
//   x = allowed ? x : -inf
// and one rounding to the logits' type.  Logits that no rule touches are copied bit for bit.
//
// Bound: HBM, logits in and out once.  A CTA takes a slice of the vocabulary for one row, or for several rows of a batch of trees: it
// counts the request's history into shared memory (all of it is read, the tokens of the slice count), marks the touched tokens in a
// bitmap and walks the slice in 16-byte vectors, of which only those with a marked or forbidden token are unpacked.  No counts
// live in memory between calls: the state of a request is the list of its tokens.
// ---------------------------------------------------------------------------
constexpr int AL_THREADS = 512;
constexpr int AL_SLICE = 8192;                       // tokens of the vocabulary per CTA
constexpr int AL_WORDS = AL_SLICE / 32 + 1;          // bitmaps, with a word past the end for reads across words
constexpr uint32_t AL_PROMPT = 0x80000000u;          // in a count: the token occurs in the prompt

struct LogitArgs {
  const void* logits;
  void* out;
  int64_t ld, ld_out;
  int rows, vocab, n_seqs, rows_per_cta;
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
};

template <class T>
struct Logit;
template <>
struct Logit<uint16_t> {
  static constexpr uint16_t kMinusInf = 0xff80;
  static __device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};
template <>
struct Logit<uint32_t> {
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static __device__ __forceinline__ float widen(uint32_t x) { return __uint_as_float(x); }
  static __device__ __forceinline__ uint32_t narrow(float x) { return __float_as_uint(x); }
};

// n <= 8 bits of a bitmap from bit i on
__device__ __forceinline__ uint32_t bits_at(const uint32_t* map, int i, int n) {
  return __funnelshift_r(map[i >> 5], map[(i >> 5) + 1], i & 31) & ((1u << n) - 1);
}

template <class T>
__global__ void __launch_bounds__(AL_THREADS) adjust_logits_kernel(const LogitArgs a) {
  extern __shared__ uint32_t s_counts[];  // [AL_SLICE], then the same of places in the request's list of biases, from 1
  uint32_t* const s_bias = s_counts + AL_SLICE;
  __shared__ uint32_t s_touched[AL_WORDS], s_allowed[AL_WORDS];
  constexpr int V = 16 / sizeof(T), PER = AL_SLICE / (V * AL_THREADS);
  const int tid = threadIdx.x, v0 = blockIdx.x * AL_SLICE, len = min(AL_SLICE, a.vocab - v0);
  b2::pdl_launch_dependents();
  b2::pdl_wait();

  int seq = -1, node0 = 0, nodes = 0;
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  const int row0 = blockIdx.y * a.rows_per_cta, row1 = min(a.rows, row0 + a.rows_per_cta);
  for (int row = row0; row < row1; ++row) {
    const T* in = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.ld + v0;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.ld_out + v0;
    // 16-byte vectors where both rows allow them, the elements before and behind one by one
    const bool same = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int head = same ? min(len, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / static_cast<int>(sizeof(T))) : len;
    const int vectors = (len - head) / V;
    uint4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * AL_THREADS + tid < vectors) x[i] = *reinterpret_cast<const uint4*>(in + head + (i * AL_THREADS + tid) * V);

    // ---- the row's request ----
    int s = row;
    if (a.cu != nullptr) {
      int lo = 0, hi = a.n_seqs;  // the first request whose rows end behind this one
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(a.cu + mid + 1) > row) hi = mid;
        else lo = mid + 1;
      }
      s = lo;
    }
    const bool ruled = s < a.n_seqs;  // rows behind the last request are copied
    __syncthreads();                  // (the row before is done with the shared arrays)
    if (ruled && s != seq) {
      for (int i = tid; i < AL_SLICE; i += AL_THREADS) {
        s_counts[i] = 0;
        if (a.n_bias > 0) s_bias[i] = 0;
      }
      for (int i = tid; i < AL_WORDS; i += AL_THREADS) s_touched[i] = 0;
      __syncthreads();
      if (a.history != nullptr) {
        const int64_t* text = a.history + static_cast<int64_t>(s) * a.history_stride;
        const int n = max(0, min(__ldg(a.history_lens + s), a.history_width)), prompt = a.prompt_lens != nullptr ? __ldg(a.prompt_lens + s) : 0;
        for (int i = tid; i < n; i += AL_THREADS) {
          const int64_t e = __ldg(reinterpret_cast<const long long*>(text) + i) - v0;
          if (e < 0 || e >= len) continue;
          if (i < prompt) atomicOr(s_counts + e, AL_PROMPT);
          else atomicAdd(s_counts + e, 1u);
          atomicOr(s_touched + (e >> 5), 1u << (e & 31));
        }
      }
      for (int i = tid; i < a.n_bias; i += AL_THREADS) {
        const int64_t e = __ldg(reinterpret_cast<const long long*>(a.bias_ids) + s * a.bias_stride + i) - v0;
        if (e < 0 || e >= len) continue;
        atomicMax(s_bias + e, static_cast<uint32_t>(i + 1));
        atomicOr(s_touched + (e >> 5), 1u << (e & 31));
      }
      seq = s;
      repetition = a.repetition != nullptr ? __ldg(a.repetition + s) : 1.f;
      presence = a.presence != nullptr ? __ldg(a.presence + s) : 0.f;
      frequency = a.frequency != nullptr ? __ldg(a.frequency + s) : 0.f;
      if (a.cu != nullptr) {
        node0 = max(0, __ldg(a.cu + s));
        nodes = min(min(a.rows, __ldg(a.cu + s + 1)) - node0, 64 * a.words);
      }
    }
    // the drafted tokens that this row's node sees, as output; afterwards they are taken out again
    auto path = [&](int sign) {
      if (!ruled || a.drafts == nullptr) return;
      for (int k = tid; k < nodes; k += AL_THREADS) {
        if (!((__ldg(reinterpret_cast<const unsigned long long*>(a.tree_mask + static_cast<int64_t>(row) * a.mask_stride + (k >> 6))) >> (k & 63)) & 1)) continue;
        const int64_t e = __ldg(reinterpret_cast<const long long*>(a.drafts) + node0 + k) - v0;
        if (e < 0 || e >= len) continue;
        atomicAdd(s_counts + e, static_cast<uint32_t>(sign));
        if (sign > 0) atomicOr(s_touched + (e >> 5), 1u << (e & 31));  // (a mark that stays costs the next row a look at a count of zero)
      }
    };
    path(1);
    if (a.allowed != nullptr)
      for (int i = tid; i < (len + 31) / 32; i += AL_THREADS) s_allowed[i] = __ldg(a.allowed + static_cast<int64_t>(row) * a.allowed_stride + v0 / 32 + i);
    __syncthreads();

    // ---- the slice ----
    auto rule = [&](T raw, int e) -> T {
      if (a.allowed != nullptr && !((s_allowed[e >> 5] >> (e & 31)) & 1)) return Logit<T>::kMinusInf;
      if (!((s_touched[e >> 5] >> (e & 31)) & 1)) return raw;
      const uint32_t c = s_counts[e], count = c & ~AL_PROMPT;
      float x = Logit<T>::widen(raw);
      if (c != 0 && a.repetition != nullptr) x = x > 0.f ? __fdiv_rn(x, repetition) : x * repetition;
      if (count != 0) {
        x = __fsub_rn(x, __fmul_rn(frequency, static_cast<float>(count)));
        x = __fsub_rn(x, presence);
      }
      if (a.n_bias > 0) {
        const uint32_t i = s_bias[e];
        if (i != 0) x += __ldg(a.bias_values + s * a.bias_value_stride + i - 1);
      }
      return Logit<T>::narrow(x);
    };
    auto element = [&](int e) { out[e] = ruled ? rule(in[e], e) : in[e]; };
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = i * AL_THREADS + tid;
      if (k >= vectors) break;
      const int e0 = head + k * V;
      constexpr uint32_t all = (1u << V) - 1;
      uint32_t special = ruled ? bits_at(s_touched, e0, V) : 0u;
      if (ruled && a.allowed != nullptr) special |= bits_at(s_allowed, e0, V) ^ all;
      if (special != 0) {
        T* const raw = reinterpret_cast<T*>(&x[i]);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if ((special >> e) & 1) raw[e] = rule(raw[e], e0 + e);
      }
      *reinterpret_cast<uint4*>(out + e0) = x[i];
    }
    for (int e = tid; e < head; e += AL_THREADS) element(e);
    for (int e = head + vectors * V + tid; e < len; e += AL_THREADS) element(e);
    if (row + 1 < row1 && ruled && a.drafts != nullptr) {
      __syncthreads();
      path(-1);
    }
  }
}

size_t adjust_smem(int n_bias) { return static_cast<size_t>(n_bias > 0 ? 2 : 1) * AL_SLICE * sizeof(uint32_t); }

int configure_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  B2_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return b2::set_error(B2_ERR_UNSUPPORTED, "device ordinal %d not supported", dev);
  if (!done[dev].load(std::memory_order_acquire)) {
    B2_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<uint16_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, adjust_smem(1)));
    B2_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<uint32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, adjust_smem(1)));
    done[dev].store(true, std::memory_order_release);
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
  if (r->draft_tokens != nullptr && (!r->tree_mask || !r->cu_seqlens || r->mask_words <= 0 || r->mask_stride < r->mask_words || r->mask_words > 1 << 20)) return B2_ERR_ARG;
  const int rc = configure_once();
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
  // rows of one request share the counts of its history: as many to a CTA as leave four CTAs for every SM
  const int slices = (vocab + AL_SLICE - 1) / AL_SLICE;
  a.rows_per_cta = r->cu_seqlens == nullptr ? 1 : std::max(1, static_cast<int>(static_cast<int64_t>(rows) * slices / (4 * 148)));
  a.rows_per_cta = std::max(a.rows_per_cta, (rows + 65534) / 65535);
  const dim3 grid(slices, (rows + a.rows_per_cta - 1) / a.rows_per_cta);
  const auto kernel = fp32 ? adjust_logits_kernel<uint32_t> : adjust_logits_kernel<uint16_t>;
  B2_CUDA(b2_launch(kernel, grid, dim3(AL_THREADS), adjust_smem(r->n_bias), static_cast<cudaStream_t>(stream), a));
  return B2_OK;
}
