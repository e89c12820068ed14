// Bindings of the operators around an 8-bit paged cache (rotary store, read and decode) and of decode over shared prefixes.  Rows are e4m3 (num_blocks, block_size, H_KV,
// D), their powers of two E8M0 (num_blocks, H_KV, block_size).  There is no CPU path: a tensor that is not on the GPU is an error.

#include "paged_common.h"

namespace py = pybind11;

namespace {

// One side of a cache, keys or values.
struct Side {
    uint8_t *codes, *scales;
    int64_t s[3], ss[2];            // strides {block, token, head} and {block, head}; 0 where there is one only
};
Side side_of(const at::Tensor& cache, const at::Tensor& scales, const at::Tensor& like, int64_t D) {
    check_place(cache, like, "every cache");
    check_place(scales, like, "every scale tensor");
    check(cache.dim() == 4 && cache.size(3) == D && cache.scalar_type() == at::kFloat8_e4m3fn && (cache.stride(3) == 1 || cache.size(3) <= 1),
          "key and value caches must be float8_e4m3fn of shape (num_blocks, block_size, H_KV, D) with contiguous rows");
    check(scales.dim() == 3 && scales.scalar_type() == at::kFloat8_e8m0fnu && scales.size(0) == cache.size(0) && scales.size(1) == cache.size(2) &&
              scales.size(2) == cache.size(1) && (scales.stride(2) == 1 || scales.size(2) <= 1),
          "key and value scales must be float8_e8m0fnu of shape (num_blocks, H_KV, block_size) with the tokens of a page contiguous");
    Side r = {static_cast<uint8_t*>(cache.data_ptr()), static_cast<uint8_t*>(scales.data_ptr()), {}, {}};
    for (int i = 0; i < 3; ++i) r.s[i] = cache.size(i) > 1 ? cache.stride(i) : 0;
    for (int i = 0; i < 2; ++i) r.ss[i] = scales.size(i) > 1 ? scales.stride(i) : 0;
    return r;
}
// Whether two tensors of one layout, some bytes apart, share none although their extents meet (rows side by side in the records of pages):
// from the largest stride down, indices of a dimension have to be equal where all that lies within it, of both, fits its stride.
bool alike_and_apart(const at::Tensor& a, const at::Tensor& b) {
    if (a.sizes() != b.sizes() || a.strides() != b.strides() || a.element_size() != 1 || b.element_size() != 1) return false;
    const int64_t between = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
    const int64_t apart = between < 0 ? -between : between;
    uint32_t left = 0;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1) left |= 1u << i;
    for (;;) {
        int64_t span = 1, largest = -1;
        for (int64_t i = 0; i < a.dim(); ++i) {
            if ((left >> i & 1) == 0) continue;
            span += (a.size(i) - 1) * a.stride(i);
            if (largest < 0 || a.stride(i) > a.stride(largest)) largest = i;
        }
        if (span <= apart) return true;
        if (largest < 0) return false;
        const int64_t within = span - (a.size(largest) - 1) * a.stride(largest);
        if (apart + within > a.stride(largest)) return false;
        left &= ~(1u << largest);
    }
}
void check_alike(const at::Tensor& key_cache, const at::Tensor& value_cache) {
    check(key_cache.sizes() == value_cache.sizes(), "the caches must have one shape");
}

at::Tensor rotary_paged_store8(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& positions,
                               const at::Tensor& slot_mapping, const at::Tensor& inv_freq, at::Tensor key_cache, at::Tensor value_cache,
                               at::Tensor key_scales, at::Tensor value_scales, bool interleaved, double scale, const MaybeTensor& out) {
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
    const Side ks = side_of(key_cache, key_scales, q, q.size(2)), vs = side_of(value_cache, value_scales, q, q.size(2));
    check_alike(key_cache, value_cache);
    check(key_cache.size(2) == k.size(1), "the caches must have the heads of k");
    const at::Tensor* const kept[] = {&key_cache, &value_cache, &key_scales, &value_scales};
    for (int i = 0; i < 4; ++i) {
        check(!rows_meet(*kept[i]), "rows of a cache must not share memory");
        for (int j = 0; j < i; ++j) check(!caches_may_meet(*kept[i], *kept[j]) || alike_and_apart(*kept[i], *kept[j]), "keys, values and their scales must share no memory");
    }
    c10::DeviceGuard guard(q.device());
    const Angles a = angles_of(positions, inv_freq, q);
    const at::Tensor qc = rows_in(q), kc = rows_in(k), vc = rows_in(v), sm = slot_mapping.contiguous();
    const at::Tensor qo = rows_out(out, qc, q, k, "out");
    check(!out.has_value() || (!may_meet(qo, v) && !extents_meet_any(qo, {&positions, &inv_freq, &slot_mapping})),
          "out must share no memory with the other operands");
    for (const at::Tensor* c : kept) {
        check_written(*c);
        check(!extents_meet_any(*c, {&q, &k, &v, &qo, &positions, &inv_freq, &slot_mapping}), "the caches must share no memory with the other operands");
    }
    const int64_t qs[2] = {qc.stride(0), qc.stride(1)}, qos[2] = {qo.stride(0), qo.stride(1)};
    const int64_t kst[2] = {kc.stride(0), kc.stride(1)}, vst[2] = {vc.stride(0), vc.stride(1)};
    const int st = fq_rotary_paged_store8(qc.data_ptr(), qs, qo.data_ptr(), qos, int(q.size(1)), kc.data_ptr(), kst, vc.data_ptr(), vst,
                                          int(k.size(1)), a.positions.data_ptr(), a.bytes, a.inv_freq.data_ptr<double>(), a.half, interleaved,
                                          float(scale), sm.data_ptr<int64_t>(), sm.size(0), ks.codes, ks.s, vs.codes, vs.s, ks.scales, ks.ss,
                                          vs.scales, vs.ss, int(key_cache.size(1)), key_cache.size(0), q.size(0), int(q.size(2)),
                                          fqbind::dtype_code(q.scalar_type(), "rotary_paged_store8"), fqbind::current_stream(q));
    fqbind::raise_on_error(st, "rotary_paged_store8");
    for (const at::Tensor* c : kept) written(*c);
    if (out.has_value()) written(qo);
    return qo;
}

std::tuple<at::Tensor, at::Tensor> paged_kv8_read(const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& key_scales,
                                                  const at::Tensor& value_scales, const at::Tensor& block_table, const at::Tensor& cu_seqlens,
                                                  int64_t num_tokens, const MaybeTensor& starts, at::ScalarType dtype,
                                                  const std::optional<std::tuple<at::Tensor, at::Tensor>>& out) {
    fqbind::require_gpu(key_cache, "key_cache");
    check(key_cache.dim() == 4, "key and value caches must be float8_e4m3fn of shape (num_blocks, block_size, H_KV, D) with contiguous rows");
    const int64_t H = key_cache.size(2), D = key_cache.size(3);
    const Side ks = side_of(key_cache, key_scales, key_cache, D), vs = side_of(value_cache, value_scales, key_cache, D);
    check_alike(key_cache, value_cache);
    check_place(block_table, key_cache, "block_table");
    check_place(cu_seqlens, key_cache, "cu_seqlens");
    check(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && (block_table.stride(1) == 1 || block_table.size(1) <= 1),
          "block_table must be int32 of shape (num_seqs, max_blocks) with contiguous rows");
    const int64_t S = block_table.size(0);
    check(cu_seqlens.dim() == 1 && cu_seqlens.scalar_type() == at::kInt && cu_seqlens.size(0) == S + 1, "cu_seqlens must be int32 of shape (num_seqs + 1,)");
    if (starts.has_value()) {
        check_place(*starts, key_cache, "starts");
        check(starts->dim() == 1 && starts->scalar_type() == at::kInt && starts->size(0) == S, "starts must be int32 of shape (num_seqs,)");
    }
    check(dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be float16 or bfloat16");
    check(num_tokens >= 0 && num_tokens <= 0x7fffffff, "num_tokens must be >= 0 and below 2^31");
    check(S <= (1 << 30) && block_table.size(1) <= 0x7fffffff && H <= 4096 && D <= 4096, "too large a size");
    c10::DeviceGuard guard(key_cache.device());
    const at::Tensor cu = cu_seqlens.contiguous(), first = starts.has_value() ? starts->contiguous() : at::Tensor();
    at::Tensor keys, values;
    if (out.has_value()) {
        std::tie(keys, values) = *out;
        for (const at::Tensor* t : {&keys, &values}) {
            check_place(*t, key_cache, "out");
            check(t->is_contiguous() && t->scalar_type() == dtype && t->dim() == 3 && t->size(0) == num_tokens && t->size(1) == H && t->size(2) == D,
                  "out must be two contiguous tensors of shape (num_tokens, H_KV, D) and of dtype");
            check(!extents_meet_any(*t, {&key_cache, &value_cache, &key_scales, &value_scales, &block_table, &cu_seqlens, starts.has_value() ? &*starts : &cu_seqlens}),
                  "out must share no memory with the inputs");
            check_written(*t);
        }
        check(!extents_meet_any(keys, {&values}), "the outputs must share no memory");
    } else {
        keys = new_tensor({num_tokens, H, D}, dtype, key_cache);
        values = new_tensor({num_tokens, H, D}, dtype, key_cache);
    }
    if (num_tokens == 0 || H == 0) return {keys, values};
    const int st = fq_paged_kv8_read(ks.codes, ks.s, vs.codes, vs.s, ks.scales, ks.ss, vs.scales, vs.ss, block_table.data_ptr<int32_t>(),
                                     block_table.stride(0), cu.data_ptr<int32_t>(), first.defined() ? first.data_ptr<int32_t>() : nullptr,
                                     keys.data_ptr(), values.data_ptr(), out.has_value() ? 0 : 1, int(S), num_tokens, int(H), int(D),
                                     int(key_cache.size(1)), int(block_table.size(1)), key_cache.size(0), fqbind::dtype_code(dtype, "paged_kv8_read"),
                                     fqbind::current_stream(key_cache));
    fqbind::raise_on_error(st, "paged_kv8_read");
    if (out.has_value()) {
        written(keys);
        written(values);
    }
    return {keys, values};
}

// What the decodes check and make alike: the query as the kernels take it, the result, room.
struct DecodeCall {
    at::Tensor q, lens, out, lse, ws;
    int64_t S, HQ, HKV, D;
    int block_size, max_blocks;
};
void check_decode(DecodeCall& c, const at::Tensor& q, const at::Tensor& key_cache, const at::Tensor& block_table, const at::Tensor& seq_lens) {
    check_place(block_table, q, "block_table");
    check_place(seq_lens, q, "seq_lens");
    c.S = q.size(0); c.HQ = q.size(1); c.D = q.size(2); c.HKV = key_cache.size(2);
    check(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && block_table.size(0) == c.S &&
              (block_table.stride(1) == 1 || block_table.size(1) <= 1),
          "block_table must be int32 of shape (num_seqs, max_blocks) with contiguous rows");
    check(seq_lens.dim() == 1 && seq_lens.scalar_type() == at::kInt && seq_lens.size(0) == c.S, "seq_lens must be int32 of shape (num_seqs,)");
    check(c.S <= 0x7fffffff && c.HQ <= 0x7fffffff && c.HKV <= 0x7fffffff && block_table.size(1) <= 0x7fffffff && key_cache.size(1) <= 0x7fffffff, "too large a size");
    c.block_size = int(key_cache.size(1));
    c.max_blocks = int(block_table.size(1));
}
void set_up_decode(DecodeCall& c, const at::Tensor& q, const at::Tensor& seq_lens, std::initializer_list<const at::Tensor*> inputs, const MaybeTensor& out,
                   bool return_lse, size_t bytes, const MaybeTensor& workspace, const char* too_small) {
    c.q = rows_in(q);
    if (reinterpret_cast<uintptr_t>(c.q.data_ptr()) % 16 != 0 || c.q.stride(0) % 8 != 0 || c.q.stride(1) % 8 != 0)
        c.q = c.q.clone(at::MemoryFormat::Contiguous);
    c.lens = seq_lens.contiguous();
    if (out.has_value()) {
        c.out = *out;
        check_place(c.out, q, "out");
        check(c.out.is_contiguous() && c.out.scalar_type() == q.scalar_type() && c.out.sizes() == q.sizes(),
              "out must be a contiguous GPU tensor with the shape and dtype of q");
        check(!may_meet(c.out, q) && !extents_meet_any(c.out, inputs), "out must share no memory with the inputs");
        check_written(c.out);
    } else {
        c.out = new_tensor(q.sizes(), q.scalar_type(), q);
    }
    if (return_lse) c.lse = new_tensor({c.S, c.HQ}, at::kFloat, q);
    if (workspace.has_value()) {
        c.ws = *workspace;
        check_place(c.ws, q, "workspace");
        check(c.ws.is_contiguous() && c.ws.scalar_type() == at::kByte && size_t(c.ws.numel()) >= bytes, too_small);
        check(!extents_meet_any(c.ws, inputs) && !extents_meet_any(c.ws, {&q, &c.out}), "workspace must share no memory with the operands");
    } else if (bytes > 0) {
        c.ws = new_tensor({int64_t(bytes)}, at::kByte, q);
    }
}

std::tuple<at::Tensor, MaybeTensor> paged_kv8_decode(const at::Tensor& q, const at::Tensor& key_cache, const at::Tensor& value_cache,
                                                     const at::Tensor& key_scales, const at::Tensor& value_scales, const at::Tensor& block_table,
                                                     const at::Tensor& seq_lens, double sm_scale, int64_t window, const MaybeTensor& out,
                                                     bool return_lse, const MaybeTensor& workspace) {
    fqbind::require_gpu(q, "q");
    check(q.dim() == 3 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16), "q must be float16 or bfloat16 of shape (num_seqs, H_Q, D)");
    const Side ks = side_of(key_cache, key_scales, q, q.size(2)), vs = side_of(value_cache, value_scales, q, q.size(2));
    check_alike(key_cache, value_cache);
    DecodeCall c;
    check_decode(c, q, key_cache, block_table, seq_lens);
    check(window >= 0 && window <= 0x7fffffff, "window must be >= 0");
    c10::DeviceGuard guard(q.device());
    const size_t bytes = fq_paged_kv8_decode_workspace_needed(int(c.S), int(c.HQ), int(c.HKV), int(c.D), c.block_size, c.max_blocks, int(window));
    set_up_decode(c, q, seq_lens, {&key_cache, &value_cache, &key_scales, &value_scales, &block_table, &seq_lens}, out, return_lse, bytes, workspace,
                  "workspace must be a contiguous uint8 GPU tensor of at least paged_kv8_decode_workspace_bytes(...) bytes");
    const int64_t qs[2] = {c.q.stride(0), c.q.stride(1)};
    const int st = fq_paged_kv8_decode(c.q.data_ptr(), qs, ks.codes, ks.s, vs.codes, vs.s, ks.scales, ks.ss, vs.scales, vs.ss,
                                       block_table.data_ptr<int32_t>(), block_table.stride(0), c.lens.data_ptr<int32_t>(), c.out.data_ptr(),
                                       return_lse ? c.lse.data_ptr<float>() : nullptr, int(c.S), int(c.HQ), int(c.HKV), int(c.D), c.block_size,
                                       c.max_blocks, key_cache.size(0), float(sm_scale), int(window),
                                       fqbind::dtype_code(q.scalar_type(), "paged_kv8_decode"), c.ws.defined() ? c.ws.data_ptr() : nullptr,
                                       c.ws.defined() ? size_t(c.ws.numel()) : 0, fqbind::current_stream(q));
    fqbind::raise_on_error(st, "paged_kv8_decode");
    if (out.has_value()) written(c.out);
    return {c.out, return_lse ? MaybeTensor(c.lse) : std::nullopt};
}

// 16-bit caches, or 8-bit ones with their scales
std::tuple<at::Tensor, MaybeTensor> paged_prefix_decode(const at::Tensor& q, const at::Tensor& key_cache, const at::Tensor& value_cache,
                                                        const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& prefix_ids,
                                                        const at::Tensor& prefix_lens, double sm_scale, const MaybeTensor& key_scales,
                                                        const MaybeTensor& value_scales, const MaybeTensor& out, bool return_lse,
                                                        const MaybeTensor& workspace) {
    fqbind::require_gpu(q, "q");
    check(q.dim() == 3 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16), "q must be float16 or bfloat16 of shape (num_seqs, H_Q, D)");
    check(key_scales.has_value() == value_scales.has_value(), "key_scales and value_scales belong together");
    const bool f8 = key_scales.has_value();
    Side ks = {}, vs = {};
    if (f8) {
        ks = side_of(key_cache, *key_scales, q, q.size(2));
        vs = side_of(value_cache, *value_scales, q, q.size(2));
    } else {
        const Cache k = cache_of(key_cache, q, q, "key_cache"), v = cache_of(value_cache, q, q, "value_cache");
        for (int i = 0; i < 3; ++i) {
            ks.s[i] = key_cache.size(i) > 1 ? k.s[i] : 0;
            vs.s[i] = value_cache.size(i) > 1 ? v.s[i] : 0;
        }
    }
    check_alike(key_cache, value_cache);
    DecodeCall c;
    check_decode(c, q, key_cache, block_table, seq_lens);
    check_place(prefix_ids, q, "prefix_ids");
    check_place(prefix_lens, q, "prefix_lens");
    check(prefix_ids.dim() == 1 && prefix_ids.scalar_type() == at::kInt && prefix_ids.size(0) == c.S, "prefix_ids must be int32 of shape (num_seqs,)");
    check(prefix_lens.dim() == 1 && prefix_lens.scalar_type() == at::kInt && prefix_lens.size(0) <= 1024,
          "prefix_lens must be int32 of one dimension, of 1024 prefixes at most");
    c10::DeviceGuard guard(q.device());
    const at::Tensor ids = prefix_ids.contiguous(), lens = prefix_lens.contiguous();
    const size_t bytes = fq_paged_prefix_decode_workspace_bytes(int(c.S), int(c.HQ), int(c.HKV), int(c.D), int(lens.size(0)));
    set_up_decode(c, q, seq_lens,
                  {&key_cache, &value_cache, f8 ? &*key_scales : &key_cache, f8 ? &*value_scales : &value_cache, &block_table, &seq_lens, &prefix_ids, &prefix_lens},
                  out, return_lse, bytes, workspace, "workspace must be a contiguous uint8 GPU tensor of at least paged_prefix_decode_workspace_bytes(...) bytes");
    const int64_t qs[2] = {c.q.stride(0), c.q.stride(1)};
    const int st = fq_paged_prefix_decode(c.q.data_ptr(), qs, key_cache.data_ptr(), ks.s, value_cache.data_ptr(), vs.s, ks.scales, ks.ss, vs.scales, vs.ss,
                                          block_table.data_ptr<int32_t>(), block_table.stride(0), c.lens.data_ptr<int32_t>(),
                                          ids.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), int(lens.size(0)), c.out.data_ptr(),
                                          return_lse ? c.lse.data_ptr<float>() : nullptr, int(c.S), int(c.HQ), int(c.HKV), int(c.D), c.block_size,
                                          c.max_blocks, key_cache.size(0), float(sm_scale), fqbind::dtype_code(q.scalar_type(), "paged_prefix_decode"),
                                          c.ws.defined() ? c.ws.data_ptr() : nullptr, c.ws.defined() ? size_t(c.ws.numel()) : 0,
                                          fqbind::current_stream(q));
    fqbind::raise_on_error(st, "paged_prefix_decode");
    if (out.has_value()) written(c.out);
    return {c.out, return_lse ? MaybeTensor(c.lse) : std::nullopt};
}

}  // namespace

void bind_paged_kv8(py::module_& m) {
    m.def("rotary_paged_store8", &rotary_paged_store8, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("positions"), py::arg("slot_mapping"),
          py::arg("inv_freq"), py::arg("key_cache"), py::arg("value_cache"), py::arg("key_scales"), py::arg("value_scales"),
          py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("out") = py::none(),
          "Rotary positions on q and k; k and v quantised into their slots of an 8-bit paged cache; the rotated q");
    m.def("paged_kv8_read", &paged_kv8_read, py::arg("key_cache"), py::arg("value_cache"), py::arg("key_scales"), py::arg("value_scales"),
          py::arg("block_table"), py::arg("cu_seqlens"), py::arg("num_tokens"), py::arg("starts") = py::none(),
          py::arg("dtype") = at::kBFloat16, py::arg("out") = py::none(), "Tokens of an 8-bit paged cache as 16-bit rows: (keys, values)");
    m.def("paged_kv8_decode", &paged_kv8_decode, py::arg("q"), py::arg("key_cache"), py::arg("value_cache"), py::arg("key_scales"),
          py::arg("value_scales"), py::arg("block_table"), py::arg("seq_lens"), py::arg("sm_scale"), py::arg("window") = 0,
          py::arg("out") = py::none(), py::arg("return_lse") = false, py::arg("workspace") = py::none(),
          "Attention of one query per sequence over an 8-bit paged cache: (out, lse or None)");
    m.def("paged_kv8_decode_workspace_bytes", &fq_paged_kv8_decode_workspace_bytes, py::arg("num_seqs"), py::arg("H_Q"), py::arg("H_KV"),
          py::arg("head_dim"), py::arg("block_size"), py::arg("max_blocks_per_seq"));
    m.def("paged_prefix_decode", &paged_prefix_decode, py::arg("q"), py::arg("key_cache"), py::arg("value_cache"), py::arg("block_table"),
          py::arg("seq_lens"), py::arg("prefix_ids"), py::arg("prefix_lens"), py::arg("sm_scale"), py::arg("key_scales") = py::none(),
          py::arg("value_scales") = py::none(), py::arg("out") = py::none(), py::arg("return_lse") = false, py::arg("workspace") = py::none(),
          "Attention of one query per sequence where sequences begin with the same pages: (out, lse or None)");
    m.def("paged_prefix_decode_workspace_bytes", &fq_paged_prefix_decode_workspace_bytes, py::arg("num_seqs"), py::arg("H_Q"), py::arg("H_KV"),
          py::arg("head_dim"), py::arg("num_prefixes"));
}
