// C ABI of the cache-maintenance operators: argument checks and launches (declared in
// include/kvssd_b200.h; kernels in rotary.cu, append.cu, weights.cu and evict.cu).
#include "../../include/kvssd_b200.h"
#include "cache_ops.cuh"

using namespace kvb;

namespace {

constexpr int kMaxHeadDim = 256;

int bad(const char* message) { return report(KVSSD_B200_ERR_INVALID_ARGUMENT, message); }

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return KVSSD_B200_OK;
  (void)cudaGetLastError();
  return report(KVSSD_B200_ERR_CUDA, what);
}

int check_elements(int dtype) {
  if (dtype != KVSSD_B200_Q_F32 && dtype != KVSSD_B200_Q_F16 && dtype != KVSSD_B200_Q_BF16)
    return bad("element type must be FP32, FP16 or BF16");
  return KVSSD_B200_OK;
}

int check_rotation(int head_dim, const void* positions, const double* frequencies, int pairs) {
  if (!positions || !frequencies) return bad("positions and frequencies must not be NULL");
  if (pairs < 1 || 2ll * pairs > head_dim)
    return bad("frequencies must hold 1 to head_dim / 2 pairs");
  return KVSSD_B200_OK;
}

int check_cache(int n_pool, int bt, int kvh, int d, int bits, int group) {
  if (bits != 2 && bits != 4) return bad("bits must be 2 or 4");
  if (n_pool < 1 || bt < 1 || kvh < 1 || d < 1 || group < 1) return bad("all dimensions must be positive");
  if (d % group) return bad("group_size must divide head_dim");
  if (group % (8 / bits)) return bad("group_size must be positive and pack-aligned");
  if (d > kMaxHeadDim) return report(KVSSD_B200_ERR_UNSUPPORTED, "head_dim > 256 is not supported");
  if (kvh > 65535) return report(KVSSD_B200_ERR_UNSUPPORTED, "more than 65535 KV heads are not supported");
  return KVSSD_B200_OK;
}

int check_places(int n_sel, int bt) {
  if (n_sel < 1) return bad("at least one block is required");
  if (static_cast<long long>(n_sel) * bt > 0x7ff00000ll)  // room for a tile or batch behind the last
    return report(KVSSD_B200_ERR_UNSUPPORTED, "more than 2^31 places are not supported");
  return KVSSD_B200_OK;
}

}  // namespace

extern "C" {

int kvssd_b200_rotary(const void* x, int dtype, long long x_token_stride, long long x_head_stride,
                      int tokens, int heads, int head_dim, const void* positions,
                      int positions_int64, const double* frequencies, int pairs, int interleaved,
                      float magnitude, void* out, long long out_token_stride,
                      long long out_head_stride, kvssd_b200_stream_t stream) {
  if (tokens < 0 || heads < 0) return bad("tokens and heads must not be negative");
  if (int st = check_elements(dtype)) return st;
  if (head_dim < 1) return bad("head_dim must be positive");
  if (head_dim > kMaxHeadDim) return report(KVSSD_B200_ERR_UNSUPPORTED, "head_dim > 256 is not supported");
  if (tokens == 0 || heads == 0) return KVSSD_B200_OK;
  if (!x || !out) return bad("tensor pointers must not be NULL");
  if (int st = check_rotation(head_dim, positions, frequencies, pairs)) return st;
  if (static_cast<long long>(heads) * head_dim > 0x1000000ll)
    return report(KVSSD_B200_ERR_UNSUPPORTED, "rows of more than 2^24 elements are not supported");
  for (const long long stride : {x_token_stride, x_head_stride, out_token_stride, out_head_stride})
    if (stride > 0x7fffffffll || stride < -0x7fffffffll)
      return report(KVSSD_B200_ERR_UNSUPPORTED, "strides of 2^31 elements or more are not supported");
  RotaryArgs a{{x, x_token_stride, x_head_stride}, out, out_token_stride, out_head_stride, dtype,
               tokens, heads, head_dim, {positions, positions_int64 ? 1 : 0}, frequencies, pairs,
               interleaved ? 1 : 0, magnitude};
  return launched(launch_rotary(a, reinterpret_cast<cudaStream_t>(stream)), "rotary launch failed");
}

int kvssd_b200_append(const void* key, const void* value, int dtype, long long key_token_stride,
                      long long key_head_stride, long long value_token_stride,
                      long long value_head_stride, int tokens, const void* slots, int slots_int64,
                      const void* positions, int positions_int64, const double* frequencies,
                      int pairs, int interleaved, float magnitude, uint8_t* packed_k,
                      uint8_t* packed_v, uint16_t* scales_k, uint16_t* scales_v,
                      int32_t* valid_tokens, int n_pool_blocks, int block_tokens, int kv_heads,
                      int head_dim, int bits, int group_size, uint16_t* key_values,
                      uint16_t* value_values, unsigned* device_status, kvssd_b200_stream_t stream) {
  if (tokens < 0) return bad("tokens must not be negative");
  if (tokens > 0x7ff00000)  // room for a CTA's tokens behind the last
    return report(KVSSD_B200_ERR_UNSUPPORTED, "more than 2^31 tokens are not supported");
  if (int st = check_elements(dtype)) return st;
  if (int st = check_cache(n_pool_blocks, block_tokens, kv_heads, head_dim, bits, group_size)) return st;
  if (frequencies)
    if (int st = check_rotation(head_dim, positions, frequencies, pairs)) return st;
  if (!key_values != !value_values) return bad("pass both value outputs, or neither");
  if (tokens == 0) return KVSSD_B200_OK;
  if (!key || !value || !slots || !packed_k || !packed_v || !scales_k || !scales_v)
    return bad("tensor pointers must not be NULL");
  AppendArgs a{{key, key_token_stride, key_head_stride},
               {value, value_token_stride, value_head_stride},
               dtype, tokens, {slots, slots_int64 ? 1 : 0}, {positions, positions_int64 ? 1 : 0},
               frequencies, pairs, interleaved ? 1 : 0, magnitude,
               {packed_k, packed_v},
               {reinterpret_cast<__half*>(scales_k), reinterpret_cast<__half*>(scales_v)},
               {reinterpret_cast<__half*>(key_values), reinterpret_cast<__half*>(value_values)},
               valid_tokens, n_pool_blocks, block_tokens, kv_heads, head_dim, bits, group_size,
               device_status};
  return launched(launch_append(a, reinterpret_cast<cudaStream_t>(stream)), "append launch failed");
}

int kvssd_b200_attention_weights_scratch_size(int queries, int n_sel_blocks, int block_tokens,
                                              int query_heads, int kv_heads, int head_dim, int bits,
                                              int group_size, size_t* bytes) {
  if (!bytes) return bad("bytes must not be NULL");
  if (int st = check_cache(1, block_tokens, kv_heads, head_dim, bits, group_size)) return st;
  if (int st = check_places(n_sel_blocks, block_tokens)) return st;
  if (queries < 1 || query_heads < 1) return bad("all dimensions must be positive");
  *bytes = weights_scratch_bytes(queries, query_heads, kv_heads, n_sel_blocks, block_tokens, head_dim, group_size);
  return KVSSD_B200_OK;
}

int kvssd_b200_attention_weights(const void* query, int query_dtype, int queries,
                                 const uint8_t* packed_k, const uint16_t* scales_k,
                                 const int32_t* valid_tokens, const int32_t* block_table,
                                 const int32_t* visible, int n_pool_blocks, int n_sel_blocks,
                                 int block_tokens, int query_heads, int kv_heads, int head_dim,
                                 int bits, int group_size, float sm_scale, int lse_given,
                                 float* lse, const float* previous, long long previous_stride,
                                 float* out, long long out_stride, void* scratch,
                                 size_t scratch_bytes, unsigned* device_status,
                                 kvssd_b200_stream_t stream) {
  if (int st = check_cache(n_pool_blocks, block_tokens, kv_heads, head_dim, bits, group_size)) return st;
  if (int st = check_places(n_sel_blocks, block_tokens)) return st;
  if (!block_table && n_sel_blocks > n_pool_blocks)
    return bad("more blocks are selected than the pool holds");
  if (queries < 1 || query_heads < 1) return bad("all dimensions must be positive");
  if (query_heads % kv_heads) return bad("query heads must be divisible by KV heads");
  if (query_dtype < KVSSD_B200_Q_F32 || query_dtype > KVSSD_B200_Q_F64) return bad("unknown query dtype");
  if (!query || !packed_k || !scales_k || !valid_tokens || !lse || !out)
    return bad("tensor pointers must not be NULL");
  if (static_cast<long long>(queries) * query_heads > 0x1000000ll)
    return report(KVSSD_B200_ERR_UNSUPPORTED, "more than 2^24 query rows are not supported");
  if (!lse_given && (!scratch || scratch_bytes < weights_scratch_bytes(queries, query_heads, kv_heads, n_sel_blocks,
                                                                       block_tokens, head_dim, group_size)))
    return report(KVSSD_B200_ERR_WORKSPACE, "scratch missing or too small");
  WeightsArgs a{query, query_dtype, queries, query_heads, packed_k,
                reinterpret_cast<const __half*>(scales_k), valid_tokens, block_table, visible,
                n_pool_blocks, n_sel_blocks, block_tokens, kv_heads, head_dim, bits, group_size,
                sm_scale, lse_given ? lse : nullptr, lse, previous, previous_stride, out, out_stride,
                static_cast<float*>(scratch),
                static_cast<long long>(scratch_bytes / (2 * sizeof(float))) / (static_cast<long long>(queries) * query_heads),
                device_status};
  return launched(launch_weights(a, reinterpret_cast<cudaStream_t>(stream)),
                  "attention weights launch failed");
}

int kvssd_b200_evict_scratch_size(int n_tokens, int keep, int kv_heads, int shared, size_t* bytes) {
  if (!bytes) return bad("bytes must not be NULL");
  if (n_tokens < 1 || keep < 0 || keep > n_tokens || kv_heads < 1) return bad("bad eviction sizes");
  *bytes = sizeof(int32_t) * evict_scratch_ints(n_tokens, shared ? 1 : kv_heads);
  return KVSSD_B200_OK;
}

int kvssd_b200_evict(const float* weights, long long weights_stride, const int32_t* positions,
                     long long positions_stride, int n_tokens, int keep, int sink,
                     long long recent_from, int shared, float* new_weights,
                     int32_t* new_positions, int columns, uint8_t* packed_k, uint8_t* packed_v,
                     uint16_t* scales_k, uint16_t* scales_v, int32_t* valid_tokens,
                     const int32_t* block_table, int n_pool_blocks, int n_sel_blocks,
                     int block_tokens, int kv_heads, int packed_dim, int groups,
                     void* scratch, size_t scratch_bytes, unsigned* device_status,
                     kvssd_b200_stream_t stream) {
  if (n_pool_blocks < 1 || block_tokens < 1 || kv_heads < 1 || packed_dim < 1 || groups < 1)
    return bad("all dimensions must be positive");
  if (kv_heads > 65535 || static_cast<long long>(kv_heads) * packed_dim > 0x1000000ll ||
      static_cast<long long>(kv_heads) * groups > 0x1000000ll)
    return report(KVSSD_B200_ERR_UNSUPPORTED, "token rows of more than 2^24 bytes are not supported");
  if (int st = check_places(n_sel_blocks, block_tokens)) return st;
  if (!block_table && n_sel_blocks > n_pool_blocks)
    return bad("more blocks are selected than the pool holds");
  if (n_tokens < 1 || static_cast<long long>(n_tokens) > static_cast<long long>(n_sel_blocks) * block_tokens)
    return bad("n_tokens must lie in the selected blocks");
  if (columns < n_tokens) return bad("weights and positions must hold n_tokens columns");
  if (keep < 1 || keep > n_tokens) return bad("keep must be 1 to n_tokens");
  if (!weights || !positions || !new_weights || !new_positions || !packed_k || !packed_v ||
      !scales_k || !scales_v || !valid_tokens)
    return bad("tensor pointers must not be NULL");
  size_t need = 0;
  if (int st = kvssd_b200_evict_scratch_size(n_tokens, keep, kv_heads, shared, &need)) return st;
  if (!scratch || scratch_bytes < need)
    return report(KVSSD_B200_ERR_WORKSPACE, "scratch missing or too small");
  const int lists = shared ? 1 : kv_heads;
  int32_t* lists_at = static_cast<int32_t*>(scratch);
  EvictArgs a{weights, weights_stride, positions, positions_stride, n_tokens, keep, columns, sink,
              recent_from, shared ? 1 : 0, new_weights, new_positions, lists_at + lists,
              lists_at + lists + static_cast<size_t>(lists) * keep, lists_at,
              reinterpret_cast<unsigned*>(lists_at + lists + static_cast<size_t>(lists) * n_tokens),
              {packed_k, packed_v},
              {reinterpret_cast<__half*>(scales_k), reinterpret_cast<__half*>(scales_v)},
              valid_tokens, block_table, n_pool_blocks, n_sel_blocks, block_tokens, kv_heads,
              packed_dim, groups, device_status};
  return launched(launch_evict(a, reinterpret_cast<cudaStream_t>(stream)), "eviction launch failed");
}

}  // extern "C"
