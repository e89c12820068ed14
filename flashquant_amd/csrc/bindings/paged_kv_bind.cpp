// Bindings of the operators around a 16-bit paged cache: page scheduling, rotary positions, rotary store, decode.
// Tensors are unwrapped, checked and handed to the C ABI on torch's current stream of their device; strided rows go in as
// they are.  There is no CPU path: a tensor that is not on the GPU is an error.

#include "paged_common.h"

namespace py = pybind11;

namespace {

std::tuple<at::Tensor, MaybeTensor> rotate(const at::Tensor& q, const MaybeTensor& k, const at::Tensor& positions, const at::Tensor& inv_freq,
                                           bool interleaved, double scale, bool inverse, const MaybeTensor& q_out, const MaybeTensor& k_out) {
    fqbind::require_gpu(q, "q");
    check(q.dim() == 3 || q.dim() == 4, "q must have shape (tokens, H, D) or (batch, tokens, H, D)");
    check(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat, "q must be float16, bfloat16 or float32");
    if (k.has_value()) {
        check_place(*k, q, "k");
        check(k->dim() == q.dim() && k->size(0) == q.size(0) && k->size(-1) == q.size(-1) && (q.dim() == 3 || k->size(1) == q.size(1)) &&
                  k->scalar_type() == q.scalar_type(),
              "k must have the tokens, head dimension and dtype of q");
    }
    check(k.has_value() || !k_out.has_value(), "an output for k without a k");
    c10::DeviceGuard guard(q.device());
    const Angles a = angles_of(positions, inv_freq, q);
    const at::Tensor qc = rows_in(q), kc = k.has_value() ? rows_in(*k) : at::Tensor();
    const at::Tensor qo = rows_out(q_out, qc, q, k, "q_out");
    at::Tensor ko;
    if (k.has_value()) {
        ko = rows_out(k_out, kc, *k, q, "k_out");
        check(!q_out.has_value() || !k_out.has_value() || !may_meet(qo, ko), "the outputs must share no memory");
    }
    for (const MaybeTensor* o : {&q_out, &k_out})
        check(!o->has_value() || !extents_meet_any(**o, {&positions, &inv_freq}), "out must share no memory with the other operands");
    const bool batched = q.dim() == 4;
    const RowStrides qs = strides_of(qc), qos = strides_of(qo);
    RowStrides ks{}, kos{};
    if (k.has_value()) { ks = strides_of(kc); kos = strides_of(ko); }
    const int64_t batch = batched ? q.size(0) : 1, tokens = q.size(batched ? 1 : 0);
    const int HQ = int(q.size(-2)), HK = k.has_value() ? int(k->size(-2)) : 0;
    if (HQ > 0 || HK > 0) {
        const int st = fq_rotary_embedding(qc.data_ptr(), qs.s, qo.data_ptr(), qos.s, HQ, HK > 0 ? kc.data_ptr() : nullptr, ks.s,
                                           HK > 0 ? ko.data_ptr() : nullptr, kos.s, HK, a.positions.data_ptr(), a.bytes, a.batch_stride,
                                           a.inv_freq.data_ptr<double>(), a.half, interleaved, float(scale), inverse, batch, tokens,
                                           int(q.size(-1)), fqbind::dtype_code(q.scalar_type(), "rotary_embedding"), fqbind::current_stream(q));
        fqbind::raise_on_error(st, "rotary_embedding");
        if (q_out.has_value()) written(qo);
        if (k_out.has_value()) written(ko);
    }
    return {qo, k.has_value() ? MaybeTensor(ko) : std::nullopt};
}

std::tuple<at::Tensor, MaybeTensor> rotate_recorded(const at::Tensor& q, const MaybeTensor& k, const at::Tensor& positions,
                                                    const at::Tensor& inv_freq, bool interleaved, double scale, bool inverse);

// The rotation is linear and its transpose the rotation by the negative angles: the gradient is the same operator, as often as it
// is asked for.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const MaybeTensor& k,
                                                  const at::Tensor& positions, const at::Tensor& inv_freq, bool interleaved, double scale,
                                                  bool inverse) {
        ctx->save_for_backward({positions, inv_freq});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["inverse"] = inverse;
        ctx->set_materialize_grads(false);
        auto [qo, ko] = rotate(q, k, positions, inv_freq, interleaved, scale, inverse, std::nullopt, std::nullopt);
        torch::autograd::variable_list r = {qo};
        if (ko.has_value()) r.push_back(*ko);
        return r;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const bool dq = grads[0].defined() && ctx->needs_input_grad(0);
        const bool dk = grads.size() > 1 && grads[1].defined() && ctx->needs_input_grad(1);
        torch::autograd::variable_list r(7);
        if (!dq && !dk) return r;
        auto [a, b] = rotate_recorded(dq ? grads[0] : grads[1], dq && dk ? MaybeTensor(grads[1]) : std::nullopt, saved[0], saved[1],
                                      ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble(),
                                      !ctx->saved_data["inverse"].toBool());
        if (dq) r[0] = a;
        if (dk) r[1] = dq ? *b : a;
        return r;
    }
};

bool needs_record(const at::Tensor& q, const MaybeTensor& k) {
    return at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad()));
}
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const MaybeTensor& t) { return t.has_value() && has_tangent(*t); }

std::tuple<at::Tensor, MaybeTensor> rotate_recorded(const at::Tensor& q, const MaybeTensor& k, const at::Tensor& positions,
                                                    const at::Tensor& inv_freq, bool interleaved, double scale, bool inverse) {
    const bool dual_q = has_tangent(q), dual_k = has_tangent(k);
    if (dual_q || dual_k) {
        // forward mode: the operator is linear, so the tangent of its result is the operator on the tangent
        auto [yq, yk] = rotate_recorded(q._fw_primal(0), k.has_value() ? MaybeTensor(k->_fw_primal(0)) : std::nullopt, positions, inv_freq,
                                        interleaved, scale, inverse);
        const auto [tq, tk] = rotate_recorded(dual_q ? q._fw_grad(0) : k->_fw_grad(0), dual_q && dual_k ? MaybeTensor(k->_fw_grad(0)) : std::nullopt,
                                              positions, inv_freq, interleaved, scale, inverse);
        if (dual_q) yq = at::_make_dual(yq, tq, 0);
        if (dual_k) yk = at::_make_dual(*yk, dual_q ? *tk : tq, 0);
        return {yq, yk};
    }
    if (!needs_record(q, k)) return rotate(q, k, positions, inv_freq, interleaved, scale, inverse, std::nullopt, std::nullopt);
    const auto r = RotaryFunction::apply(q, k, positions, inv_freq, interleaved, scale, inverse);
    return {r[0], r.size() > 1 ? MaybeTensor(r[1]) : std::nullopt};
}

std::tuple<at::Tensor, MaybeTensor> rotary_embedding(const at::Tensor& q, const MaybeTensor& k, const at::Tensor& positions,
                                                     const at::Tensor& inv_freq, bool interleaved, double scale, bool inverse,
                                                     const MaybeTensor& q_out, const MaybeTensor& k_out) {
    if (!needs_record(q, k) && !has_tangent(q) && !has_tangent(k))
        return rotate(q, k, positions, inv_freq, interleaved, scale, inverse, q_out, k_out);
    check(!q_out.has_value() && !k_out.has_value(), "out cannot be combined with gradients");
    return rotate_recorded(q, k, positions, inv_freq, interleaved, scale, inverse);
}

at::Tensor rotary_paged_store(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& positions,
                              const at::Tensor& slot_mapping, const at::Tensor& inv_freq, at::Tensor key_cache, at::Tensor value_cache,
                              bool interleaved, double scale, const MaybeTensor& out) {
    fqbind::require_gpu(q, "q");
    check_place(k, q, "k");
    check_place(v, q, "v");
    check_place(slot_mapping, q, "slot_mapping");
    check(q.dim() == 3 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16), "q must be float16 or bfloat16 of shape (tokens, H_Q, D)");
    check(k.dim() == 3 && k.size(0) == q.size(0) && k.size(1) > 0 && k.size(2) == q.size(2) && k.scalar_type() == q.scalar_type() &&
              v.sizes() == k.sizes() && v.scalar_type() == q.scalar_type(),
          "k and v must have shape (tokens, H_KV, D) and the dtype of q");
    check(slot_mapping.dim() == 1 && slot_mapping.scalar_type() == at::kLong && slot_mapping.size(0) <= q.size(0),
          "slot_mapping must be int64 with at most one entry per token");
    const Cache ks = cache_of(key_cache, q, k, "key_cache"), vs = cache_of(value_cache, q, k, "value_cache");
    check(key_cache.size(2) == k.size(1) && value_cache.sizes() == key_cache.sizes(), "the caches must have one shape, with the heads of k");
    check(!rows_meet(key_cache) && !rows_meet(value_cache), "rows of a cache must not share memory");
    c10::DeviceGuard guard(q.device());
    const Angles a = angles_of(positions, inv_freq, q);
    const at::Tensor qc = rows_in(q), kc = rows_in(k), vc = rows_in(v), sm = slot_mapping.contiguous();
    const at::Tensor qo = rows_out(out, qc, q, k, "out");
    check(!out.has_value() || (!may_meet(qo, v) && !extents_meet_any(qo, {&positions, &inv_freq, &slot_mapping})),
          "out must share no memory with the other operands");
    check_written(key_cache);
    check_written(value_cache);
    const Extent keys(key_cache), values(value_cache);
    for (const at::Tensor* t : {&q, &k, &v, &qo, &positions, &inv_freq, &slot_mapping}) {
        const Extent e(*t);
        check(!e.meets(keys) && !e.meets(values), "the caches must share no memory with the other operands");
    }
    check(!caches_may_meet(key_cache, value_cache), "keys and values must have a cache each, and share no memory");
    const int64_t qs[2] = {qc.stride(0), qc.stride(1)}, qos[2] = {qo.stride(0), qo.stride(1)};
    const int64_t kst[2] = {kc.stride(0), kc.stride(1)}, vst[2] = {vc.stride(0), vc.stride(1)};
    const int st = fq_rotary_paged_store(qc.data_ptr(), qs, qo.data_ptr(), qos, int(q.size(1)), kc.data_ptr(), kst, vc.data_ptr(), vst,
                                         int(k.size(1)), a.positions.data_ptr(), a.bytes, a.inv_freq.data_ptr<double>(), a.half, interleaved,
                                         float(scale), sm.data_ptr<int64_t>(), sm.size(0), key_cache.data_ptr(), ks.s, value_cache.data_ptr(),
                                         vs.s, int(key_cache.size(1)), key_cache.size(0), q.size(0), int(q.size(2)),
                                         fqbind::dtype_code(q.scalar_type(), "rotary_paged_store"), fqbind::current_stream(q));
    fqbind::raise_on_error(st, "rotary_paged_store");
    written(key_cache);
    written(value_cache);
    if (out.has_value()) written(qo);
    return qo;
}

// (slot_mapping, positions, seq_lens, cu_seqlens, free_end); block_table is written in place
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> paged_schedule(
    const at::Tensor& context_lens, const at::Tensor& query_lens, at::Tensor block_table, const at::Tensor& free_blocks, int64_t block_size,
    int64_t num_tokens, const MaybeTensor& free_start, const std::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>>& out,
    bool capped) {
    fqbind::require_gpu(context_lens, "context_lens");
    check_place(query_lens, context_lens, "query_lens");
    check_place(block_table, context_lens, "block_table");
    check_place(free_blocks, context_lens, "free_blocks");
    const int64_t S = context_lens.numel();
    auto ints = [](const at::Tensor& t, int64_t n) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(); };
    check(ints(context_lens, S) && ints(query_lens, S), "context_lens and query_lens must be contiguous int32 of shape (num_reqs,)");
    check(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) == S && block_table.size(1) > 0 &&
              block_table.stride(1) == 1 && (S <= 1 || block_table.stride(0) >= block_table.size(1)),
          "block_table must be int32 of shape (num_reqs, max_blocks) with contiguous rows");
    check(ints(free_blocks, free_blocks.numel()), "free_blocks must be contiguous int32 of one dimension");
    check(num_tokens >= 0 && num_tokens <= 0x7fffffff, "num_tokens must be >= 0 and below 2^31");
    check(S <= 0x7fffffff - 1 && block_table.size(1) <= 0x7fffffff, "too many requests or pages");
    if (free_start.has_value()) {
        check_place(*free_start, context_lens, "free_start");
        check(free_start->scalar_type() == at::kInt && free_start->numel() == 1, "free_start must be one int32");
    }
    check_written(block_table);
    check(!extents_meet_any(block_table, {&context_lens, &query_lens, &free_blocks, free_start.has_value() ? &*free_start : &free_blocks}),
          "block_table must share no memory with the other inputs");
    c10::DeviceGuard guard(context_lens.device());
    at::Tensor slots, positions, lens, cu, end;
    if (out.has_value()) {
        std::tie(slots, positions, lens, cu, end) = *out;
        for (const at::Tensor* t : {&slots, &positions, &lens, &cu, &end}) check_place(*t, context_lens, "out");
        auto longs = [&](const at::Tensor& t) { return t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == num_tokens && t.is_contiguous(); };
        check(longs(slots) && longs(positions) && ints(lens, S) && ints(cu, S + 1) && ints(end, 1),
              "out must be what a call with these sizes returns: int64 slots and positions (num_tokens,), int32 seq_lens (num_reqs,), "
              "cu_seqlens (num_reqs + 1,) and free_end (1,)");
        const at::Tensor* const outputs[] = {&slots, &positions, &lens, &cu, &end};
        const at::Tensor* const read[] = {&context_lens, &query_lens, &free_blocks, free_start.has_value() ? &*free_start : &free_blocks, &block_table};
        for (int i = 0; i < 5; ++i) {
            check_written(*outputs[i]);
            for (const at::Tensor* r : read) check(!Extent(*outputs[i]).meets(Extent(*r)), "outputs must share no memory with inputs");
            for (int j = 0; j < i; ++j) check(!Extent(*outputs[i]).meets(Extent(*outputs[j])), "outputs must share no memory with each other");
        }
    } else {
        slots = new_tensor({num_tokens}, at::kLong, context_lens);
        positions = new_tensor({num_tokens}, at::kLong, context_lens);
        lens = new_tensor({S}, at::kInt, context_lens);
        cu = new_tensor({S + 1}, at::kInt, context_lens);
        end = new_tensor({1}, at::kInt, context_lens);
    }
    const int64_t row = S <= 1 ? block_table.size(1) : block_table.stride(0);
    const int st = (capped ? fq_paged_schedule_capped : fq_paged_schedule)(
        context_lens.data_ptr<int32_t>(), query_lens.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(), row, free_blocks.data_ptr<int32_t>(),
        free_blocks.numel(), free_start.has_value() ? free_start->data_ptr<int32_t>() : nullptr, end.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
        positions.data_ptr<int64_t>(), lens.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), int(S), num_tokens, int(block_table.size(1)),
        int(block_size), fqbind::current_stream(context_lens));
    fqbind::raise_on_error(st, "paged_schedule");
    written(block_table);
    if (out.has_value())
        for (const at::Tensor* t : {&slots, &positions, &lens, &cu, &end}) written(*t);
    return {slots, positions, lens, cu, end};
}

using Schedule = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

// (token_table, token_lens, token_prefix) where rows are asked for, the last with prefix_ids; context_lens and free_start are written in
// place.  `schedule`: what paged_schedule returned, for the same block table.
std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> advance(const Schedule& schedule, at::Tensor context_lens, at::Tensor free_start,
                                                          const at::Tensor& block_table, int64_t num_blocks, int64_t block_size, bool rows,
                                                          const MaybeTensor& prefix_ids) {
    const auto& [slots, positions, lens, cu, end] = schedule;
    fqbind::require_gpu(context_lens, "context_lens");
    for (const at::Tensor* t : {&slots, &positions, &lens, &cu, &end, static_cast<const at::Tensor*>(&free_start), &block_table})
        check_place(*t, context_lens, "every operand");
    const int64_t S = context_lens.numel(), tokens = positions.numel();
    auto is = [](const at::Tensor& t, at::ScalarType type, int64_t n) { return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous(); };
    check(is(context_lens, at::kInt, S) && is(free_start, at::kInt, 1), "context_lens must be contiguous int32 of shape (num_reqs,), free_start (1,)");
    check(is(positions, at::kLong, tokens) && is(lens, at::kInt, S) && is(cu, at::kInt, S + 1) && is(end, at::kInt, 1), "schedule must be what paged_schedule returned");
    check(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) == S && block_table.size(1) > 0 &&
              block_table.size(1) <= 0x7fffffff && block_table.stride(1) == 1 && (S <= 1 || block_table.stride(0) >= block_table.size(1)),
          "block_table must be int32 of shape (num_reqs, max_blocks) with contiguous rows");
    check(num_blocks >= 0 && num_blocks <= 0x7fffffff && S <= 0x7fffffff, "too many pages or requests");
    if (prefix_ids.has_value()) {
        check_place(*prefix_ids, context_lens, "prefix_ids");
        check(is(*prefix_ids, at::kInt, S), "prefix_ids must be contiguous int32 of shape (num_reqs,)");
        check(!extents_meet_any(*prefix_ids, {&context_lens, &free_start}), "context_lens and free_start must share no memory with the other operands");
    }
    check_written(context_lens);
    check_written(free_start);
    check(!extents_meet_any(context_lens, {&positions, &lens, &cu, &end, &free_start, &block_table}) &&
              !extents_meet_any(free_start, {&positions, &lens, &cu, &end, &block_table}),
          "context_lens and free_start must share no memory with the other operands");
    c10::DeviceGuard guard(context_lens.device());
    at::Tensor table, token_lens, token_prefix;
    const bool prefixes = rows && prefix_ids.has_value();
    if (rows) {
        table = new_tensor({tokens, block_table.size(1)}, at::kInt, context_lens);
        token_lens = new_tensor({tokens}, at::kInt, context_lens);
    }
    if (prefixes) token_prefix = new_tensor({tokens}, at::kInt, context_lens);
    const int st = fq_paged_advance_prefix(lens.data_ptr<int32_t>(), end.data_ptr<int32_t>(), int(num_blocks), context_lens.data_ptr<int32_t>(),
                                           free_start.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), positions.data_ptr<int64_t>(),
                                           block_table.data_ptr<int32_t>(), S <= 1 ? block_table.size(1) : block_table.stride(0),
                                           prefixes ? prefix_ids->data_ptr<int32_t>() : nullptr, rows ? table.data_ptr<int32_t>() : nullptr,
                                           rows ? token_lens.data_ptr<int32_t>() : nullptr, prefixes ? token_prefix.data_ptr<int32_t>() : nullptr,
                                           int(S), rows ? tokens : 0, int(block_table.size(1)), int(block_size),
                                           fqbind::current_stream(context_lens));
    fqbind::raise_on_error(st, "paged_advance");
    written(context_lens);
    written(free_start);
    return {rows ? MaybeTensor(table) : std::nullopt, rows ? MaybeTensor(token_lens) : std::nullopt, prefixes ? MaybeTensor(token_prefix) : std::nullopt};
}
std::tuple<MaybeTensor, MaybeTensor> paged_advance(const Schedule& schedule, at::Tensor context_lens, at::Tensor free_start, const at::Tensor& block_table,
                                                   int64_t num_blocks, int64_t block_size, bool rows) {
    const auto r = advance(schedule, context_lens, free_start, block_table, num_blocks, block_size, rows, std::nullopt);
    return {std::get<0>(r), std::get<1>(r)};
}

std::tuple<at::Tensor, MaybeTensor> paged_kv_decode(const at::Tensor& q, const at::Tensor& key_cache, const at::Tensor& value_cache,
                                                    const at::Tensor& block_table, const at::Tensor& seq_lens, double sm_scale, int64_t window,
                                                    const MaybeTensor& out, bool return_lse, const MaybeTensor& workspace) {
    fqbind::require_gpu(q, "q");
    check_place(block_table, q, "block_table");
    check_place(seq_lens, q, "seq_lens");
    check(q.dim() == 3 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16), "q must be float16 or bfloat16 of shape (num_seqs, H_Q, D)");
    const Cache ks = cache_of(key_cache, q, q, "key_cache"), vs = cache_of(value_cache, q, q, "value_cache");
    check(value_cache.sizes() == key_cache.sizes(), "the caches must have one shape");
    const int64_t S = q.size(0), HQ = q.size(1), D = q.size(2), HKV = key_cache.size(2);
    check(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) == S &&
              (block_table.stride(1) == 1 || block_table.size(1) <= 1),
          "block_table must be int32 of shape (num_seqs, max_blocks) with contiguous rows");
    check(seq_lens.dim() == 1 && seq_lens.scalar_type() == at::kInt && seq_lens.size(0) == S, "seq_lens must be int32 of shape (num_seqs,)");
    check(window >= 0 && window <= 0x7fffffff, "window must be >= 0");
    check(S <= 0x7fffffff && HQ <= 0x7fffffff && D <= 0x7fffffff && block_table.size(1) <= 0x7fffffff, "too large a size");
    c10::DeviceGuard guard(q.device());
    at::Tensor qc = rows_in(q);
    if (reinterpret_cast<uintptr_t>(qc.data_ptr()) % 16 != 0 || qc.stride(0) % 8 != 0 || qc.stride(1) % 8 != 0)
        qc = qc.clone(at::MemoryFormat::Contiguous);
    const at::Tensor sl = seq_lens.contiguous();
    at::Tensor result, lse;
    if (out.has_value()) {
        result = *out;
        check_place(result, q, "out");
        check(result.is_contiguous() && result.scalar_type() == q.scalar_type() && result.sizes() == q.sizes(),
              "out must be a contiguous GPU tensor with the shape and dtype of q");
        check(!may_meet(result, qc) && !extents_meet_any(result, {&key_cache, &value_cache, &block_table, &seq_lens}),
              "out must share no memory with the inputs");
        check_written(result);
    } else {
        result = new_tensor(q.sizes(), q.scalar_type(), q);
    }
    if (return_lse) lse = new_tensor({S, HQ}, at::kFloat, q);
    const int bs = int(key_cache.size(1)), mb = int(block_table.size(1));
    const size_t bytes = fq_paged_kv_decode_workspace_needed(int(S), int(HQ), int(HKV), int(D), bs, mb, int(window));
    at::Tensor ws;
    if (workspace.has_value()) {
        ws = *workspace;
        check_place(ws, q, "workspace");
        check(ws.is_contiguous() && ws.scalar_type() == at::kByte && size_t(ws.numel()) >= bytes,
              "workspace must be a contiguous uint8 GPU tensor of at least paged_kv_decode_workspace_bytes(...) bytes");
        check(!extents_meet_any(ws, {&qc, &key_cache, &value_cache, &block_table, &seq_lens, &result}), "workspace must share no memory with the operands");
    } else if (bytes > 0) {
        ws = new_tensor({int64_t(bytes)}, at::kByte, q);
    }
    const int64_t qs[2] = {qc.stride(0), qc.stride(1)};
    const int st = fq_paged_kv_decode(qc.data_ptr(), qs, key_cache.data_ptr(), ks.s, value_cache.data_ptr(), vs.s, block_table.data_ptr<int32_t>(),
                                      block_table.stride(0), sl.data_ptr<int32_t>(), result.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
                                      int(S), int(HQ), int(HKV), int(D), bs, mb, key_cache.size(0), float(sm_scale), int(window),
                                      fqbind::dtype_code(q.scalar_type(), "paged_kv_decode"), ws.defined() ? ws.data_ptr() : nullptr,
                                      ws.defined() ? size_t(ws.numel()) : 0, fqbind::current_stream(q));
    fqbind::raise_on_error(st, "paged_kv_decode");
    if (out.has_value()) written(result);
    return {result, return_lse ? MaybeTensor(lse) : std::nullopt};
}

}  // namespace

void bind_paged_kv(py::module_& m) {
    m.def("paged_schedule", &paged_schedule, py::arg("context_lens"), py::arg("query_lens"), py::arg("block_table"), py::arg("free_blocks"),
          py::arg("block_size"), py::arg("num_tokens"), py::arg("free_start") = py::none(), py::arg("out") = py::none(),
          py::arg("capped") = false,
          "Pages, slots and positions of a step's new tokens: (slot_mapping, positions, seq_lens, cu_seqlens, free_end); block_table in place");
    m.def("paged_advance", &paged_advance, py::arg("schedule"), py::arg("context_lens"), py::arg("free_start"), py::arg("block_table"),
          py::arg("num_blocks"), py::arg("block_size"), py::arg("rows"),
          "After paged_schedule: context_lens and free_start for the next one, in place; with rows (token_table, token_lens) of its tokens");
    m.def("paged_advance_prefix", &advance, py::arg("schedule"), py::arg("context_lens"), py::arg("free_start"), py::arg("block_table"),
          py::arg("num_blocks"), py::arg("block_size"), py::arg("rows"), py::arg("prefix_ids"),
          "paged_advance with the prefix of every token as well: (token_table, token_lens, token_prefix)");
    m.def("rotary_embedding", &rotary_embedding, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"),
          py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("inverse") = false, py::arg("q_out") = py::none(),
          py::arg("k_out") = py::none(), "Rotary positions on the first 2 * len(inv_freq) coordinates of every head");
    m.def("rotary_paged_store", &rotary_paged_store, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("positions"), py::arg("slot_mapping"),
          py::arg("inv_freq"), py::arg("key_cache"), py::arg("value_cache"), py::arg("interleaved") = false, py::arg("scale") = 1.0,
          py::arg("out") = py::none(), "Rotary positions on q and k; k and v into their slots of a 16-bit paged cache; the rotated q");
    m.def("paged_kv_decode", &paged_kv_decode, py::arg("q"), py::arg("key_cache"), py::arg("value_cache"), py::arg("block_table"),
          py::arg("seq_lens"), py::arg("sm_scale"), py::arg("window") = 0, py::arg("out") = py::none(), py::arg("return_lse") = false,
          py::arg("workspace") = py::none(), "Attention of one query per sequence over a 16-bit paged cache: (out, lse or None)");
    m.def("paged_kv_decode_workspace_bytes", &fq_paged_kv_decode_workspace_bytes, py::arg("num_seqs"), py::arg("H_Q"), py::arg("H_KV"),
          py::arg("head_dim"), py::arg("block_size"), py::arg("max_blocks_per_seq"));
}
