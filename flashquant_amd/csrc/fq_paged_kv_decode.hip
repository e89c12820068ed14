// Attention of one new token per sequence over a paged cache of 16-bit keys and values: the entry points.
#include "fq_paged_kv_decode.hpp"

extern "C" size_t fq_paged_kv_decode_workspace_bytes(int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq) {
    if (check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, 1) != FQ_OK || num_seqs == 0) return 0;
    // (the calls that need none lie in bands of sizes: a caller who has room for the largest has it for all)
    const int64_t tokens = int64_t(max_blocks_per_seq) * block_size;
    if ((tokens + fq::kKvTile - 1) / fq::kKvTile <= kv_whole_tiles(D)) return 0;
    return kv_room(num_seqs, H_Q, D, kv_most_shares(H_KV)).all;
}

extern "C" size_t fq_paged_kv_decode_workspace_needed(int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq,
                                                      int window) {
    if (check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, 1) != FQ_OK || num_seqs == 0 || window < 0) return 0;
    const KvPlan plan = kv_plan(num_seqs, H_KV, D, int64_t(max_blocks_per_seq) * block_size, window);
    return kv_room(num_seqs, H_Q, D, plan.shares == 0 ? 0 : kv_most_shares(H_KV)).all;
}

extern "C" int fq_paged_kv_decode(const void* q, const int64_t* q_strides, const void* key_cache, const int64_t* key_strides,
                                  const void* value_cache, const int64_t* value_strides, const int32_t* block_table,
                                  int64_t block_table_stride, const int32_t* seq_lens, void* out, float* lse, int num_seqs, int H_Q,
                                  int H_KV, int D, int block_size, int max_blocks_per_seq, int64_t num_blocks, float sm_scale,
                                  int window, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, num_blocks);
    if (bad != FQ_OK) return bad;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (window < 0 || block_table_stride < 0) return FQ_ERR_BAD_SHAPE;
    if (num_seqs == 0) return FQ_OK;
    if (!q || !q_strides || !key_cache || !key_strides || !value_cache || !value_strides || !block_table || !seq_lens || !out)
        return FQ_ERR_NULL_POINTER;
    for (int i = 0; i < 3; ++i) {
        if (key_strides[i] % 8 != 0 || value_strides[i] % 8 != 0) return FQ_ERR_MISALIGNED;
        if (i < 2 && q_strides[i] % 8 != 0) return FQ_ERR_MISALIGNED;
    }
    if (!fq_host::aligned(q, 16) || !fq_host::aligned(key_cache, 16) || !fq_host::aligned(value_cache, 16) || !fq_host::aligned(out, 16))
        return FQ_ERR_MISALIGNED;
    KvCall call;
    const int st = set_up_call(call, q, q_strides, block_table, block_table_stride, seq_lens, out, lse, num_seqs, H_Q, H_KV, D, block_size,
                               max_blocks_per_seq, num_blocks, sm_scale, window, workspace, workspace_bytes);
    if (st != FQ_OK) return st;
    set_rows(call.p, key_cache, key_strides, value_cache, value_strides);
    return launch_kv_any<false>(call.p, call.plan, D, dtype, static_cast<hipStream_t>(stream));
}
