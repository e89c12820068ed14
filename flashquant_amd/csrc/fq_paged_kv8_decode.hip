// Attention of one new token per sequence over a paged cache of 8-bit rows: the entry points.  The kernel is that of 16-bit rows
// (fq_paged_kv_decode.hpp, which says what changes).
#include "fq_paged_kv_decode.hpp"

extern "C" size_t fq_paged_kv8_decode_workspace_bytes(int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq) {
    return fq_paged_kv_decode_workspace_bytes(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq);
}

extern "C" size_t fq_paged_kv8_decode_workspace_needed(int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq,
                                                       int window) {
    return fq_paged_kv_decode_workspace_needed(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, window);
}

extern "C" int fq_paged_kv8_decode(const void* q, const int64_t* q_strides, const uint8_t* key_cache, const int64_t* key_strides,
                                   const uint8_t* value_cache, const int64_t* value_strides, const uint8_t* key_scales,
                                   const int64_t* key_scale_strides, const uint8_t* value_scales, const int64_t* value_scale_strides,
                                   const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens, void* out, float* lse,
                                   int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq, int64_t num_blocks,
                                   float sm_scale, int window, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, num_blocks);
    if (bad != FQ_OK) return bad;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (window < 0 || block_table_stride < 0) return FQ_ERR_BAD_SHAPE;
    if (num_seqs == 0) return FQ_OK;
    if (!q || !q_strides || !key_cache || !key_strides || !value_cache || !value_strides || !key_scales || !key_scale_strides || !value_scales ||
        !value_scale_strides || !block_table || !seq_lens || !out)
        return FQ_ERR_NULL_POINTER;
    if (!codes_aligned(key_cache, key_strides, key_scales, key_scale_strides) || !codes_aligned(value_cache, value_strides, value_scales, value_scale_strides) ||
        q_strides[0] % 8 != 0 || q_strides[1] % 8 != 0 || !fq_host::aligned(q, 16) || !fq_host::aligned(out, 16))
        return FQ_ERR_MISALIGNED;
    KvCall call;
    const int st = set_up_call(call, q, q_strides, block_table, block_table_stride, seq_lens, out, lse, num_seqs, H_Q, H_KV, D, block_size,
                               max_blocks_per_seq, num_blocks, sm_scale, window, workspace, workspace_bytes);
    if (st != FQ_OK) return st;
    set_codes(call.p, key_cache, key_strides, value_cache, value_strides, key_scales, key_scale_strides, value_scales, value_scale_strides);
    return launch_kv_any<true>(call.p, call.plan, D, dtype, static_cast<hipStream_t>(stream));
}
