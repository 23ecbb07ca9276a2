// Attention of trees of drafted tokens over the paged KV cache.
#include <algorithm>

#include "b2_common.cuh"

namespace {

struct TreeArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride;
  const int32_t* tables;
  int64_t bt_stride;
  int bt_width, block_size, num_blocks;
  const int32_t *cu_q, *lens;
  const int64_t* mask;
  int64_t mask_stride;
  int words, n_seqs, tokens, nq, nkv;
  float scale_log2;
  uint16_t* out;
};

// One warp per token and query head, one key after the other.
template <int HD>
__global__ void __launch_bounds__(128) tree_attention_kernel(const TreeArgs a) {
  b2::pdl_launch_dependents();
  b2::pdl_wait();
  constexpr int D = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t warp = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int token = static_cast<int>(warp / a.nq), head = static_cast<int>(warp - static_cast<int64_t>(token) * a.nq);
  if (token >= a.tokens) return;
  int b = 0, hi = a.n_seqs;
  while (b < hi) {
    const int mid = (b + hi) >> 1;
    if (__ldg(a.cu_q + mid + 1) > token) hi = mid;
    else b = mid + 1;
  }
  uint16_t* out = a.out + (static_cast<int64_t>(token) * a.nq + head) * HD + lane * D;
  float o[D] = {}, m = -INFINITY, l = 0.f;
  if (b < a.n_seqs) {
    const int nodes = __ldg(a.cu_q + b + 1) - __ldg(a.cu_q + b), len = min(__ldg(a.lens + b), a.bt_width * a.block_size), prefix = len - nodes;
    float q[D];
    for (int d = 0; d < D; ++d) q[d] = b2::bf16_lo(a.q[token * a.q_stride + head * HD + lane * D + d]) * a.scale_log2;
    for (int key = 0; prefix >= 0 && key < len; ++key) {
      const int node = key - prefix;
      if (node >= 0 && (node >= 64 * a.words || !((a.mask[token * a.mask_stride + (node >> 6)] >> (node & 63)) & 1))) continue;
      const int block = min(max(0, __ldg(a.tables + b * a.bt_stride + key / a.block_size)), a.num_blocks - 1);  // inside the cache whatever the table holds
      const int64_t at = ((static_cast<int64_t>(block) * a.block_size + key % a.block_size) * a.nkv + head / (a.nq / a.nkv)) * HD + lane * D;
      float s = 0.f;
      for (int d = 0; d < D; ++d) s += q[d] * b2::bf16_lo(a.k[at + d]);
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      const float top = fmaxf(m, s), f = m == -INFINITY ? 0.f : exp2f(m - top), p = exp2f(s - top);
      m = top;
      l = l * f + p;
      for (int d = 0; d < D; ++d) o[d] = o[d] * f + p * b2::bf16_lo(a.v[at + d]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;  // (nothing seen: zeros)
  for (int d = 0; d < D; ++d) out[d] = static_cast<uint16_t>(b2::pack_bf16(o[d] * inv, 0.f));
}

}  // namespace

extern "C" {

int b2_tree_attention_supported(int nq, int nkv, int head_dim, int block_size) {
  return nkv > 0 && nq > 0 && nq % nkv == 0 && nq / nkv <= 128 && nkv <= 65535 && (head_dim == 64 || head_dim == 128) && block_size > 0 && block_size % 16 == 0;
}

int64_t b2_tree_attention_workspace(b2_ctx* ctx, int n_seqs, int max_q, int nq, int nkv, int head_dim, int block_size, int bt_width) {
  return 0;
}

int b2_tree_attention(b2_ctx* ctx, const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int num_blocks, int block_size,
                      const int32_t* block_tables, int64_t bt_stride, int bt_width, const int32_t* cu_q, const int32_t* context_lens, const int64_t* tree_mask,
                      int64_t mask_stride, int mask_words, int n_seqs, int max_q, int tokens, int nq, int nkv, int head_dim, float scale, void* out,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  if (ctx == nullptr || n_seqs < 0 || tokens < 0 || nq <= 0 || nkv <= 0 || max_q < 0) return B2_ERR_ARG;
  if (tokens == 0) return B2_OK;
  if (!b2_tree_attention_supported(nq, nkv, head_dim, block_size)) return B2_ERR_UNSUPPORTED;
  if (!q || !k_cache || !v_cache || !cu_q || !out || (n_seqs > 0 && (!block_tables || !context_lens || !tree_mask))) return B2_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out)) & 15)
    return B2_ERR_ARG;
  if (q_stride % 8 != 0 || q_stride < static_cast<int64_t>(nq) * head_dim || num_blocks <= 0 || bt_width <= 0 || bt_stride < bt_width || mask_words <= 0 ||
      mask_stride < mask_words)
    return B2_ERR_ARG;
  if (static_cast<int64_t>(num_blocks) * block_size >= 1ll << 31 || static_cast<int64_t>(bt_width) * block_size >= 1ll << 31) return B2_ERR_SHAPE;
  const TreeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache), q_stride, block_tables, bt_stride,
                   bt_width, block_size, num_blocks, cu_q, context_lens, tree_mask, mask_stride, mask_words, n_seqs, tokens, nq, nkv, scale * 1.4426950408889634f,
                   static_cast<uint16_t*>(out)};
  const int64_t grid = (static_cast<int64_t>(tokens) * nq + 3) / 4;
  if (grid > 0x7fffffff) return B2_ERR_SHAPE;
  B2_CUDA(b2_launch(head_dim == 128 ? tree_attention_kernel<128> : tree_attention_kernel<64>, dim3(static_cast<unsigned>(grid)), dim3(128), 0,
                    static_cast<cudaStream_t>(stream), a));
  return B2_OK;
}

}  // extern "C"
