// What the bindings of the operators around 16-bit and 8-bit paged caches share: checks of operands, new results, memory that must not meet.
#pragma once

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>

#include <optional>
#include <tuple>

#include "common.h"

namespace {

using MaybeTensor = std::optional<at::Tensor>;

// (a literal costs nothing until it is needed)
inline void check(bool ok, const char* msg) {
    if (!ok) throw std::invalid_argument(msg);
}

inline void check_place(const at::Tensor& t, const at::Tensor& like, const char* name) {
    fqbind::require_gpu(t, name);
    if (t.device() != like.device()) throw std::invalid_argument(std::string(name) + " must be on the device of the first operand");
}

// (past torch's dispatcher: half of what at::empty costs a call)
inline at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}

// rows (..., H, D) of contiguous values, as the kernels take them; others are copied
inline at::Tensor rows_in(const at::Tensor& x) { return x.stride(-1) == 1 || x.size(-1) <= 1 ? x : x.contiguous(); }

struct RowStrides {
    int64_t s[3];       // batch, token, head
};
inline RowStrides strides_of(const at::Tensor& x) {
    const int64_t n = x.dim();
    return {{n == 4 ? x.stride(0) : 0, x.stride(n - 3), x.stride(n - 2)}};
}

// The memory from a tensor's first element to its last.
struct Extent {
    const char *begin = nullptr, *end = nullptr;
    explicit Extent(const at::Tensor& t) {
        if (t.numel() == 0) return;
        const auto sizes = t.sizes(), strides = t.strides();
        int64_t last = 0;
        for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
        begin = static_cast<const char*>(t.data_ptr());
        end = begin + (last + 1) * int64_t(t.element_size());
    }
    bool meets(const Extent& o) const { return begin < o.end && o.begin < end; }        // (nothing meets no memory)
};
inline bool extents_meet_any(const at::Tensor& a, std::initializer_list<const at::Tensor*> others) {
    const Extent e(a);
    for (const at::Tensor* t : others)
        if (e.meets(Extent(*t))) return true;
    return false;
}

// Whether rows of a tensor that is written lie on each other (expanded ones, windows that slide): taken from the smallest stride up, each
// has to go past all that lies below it.
inline bool rows_meet(const at::Tensor& t) {
    if (t.is_contiguous() || t.numel() == 0) return false;
    const auto sizes = t.sizes(), strides = t.strides();
    uint32_t left = 0;                      // dimensions that are still to be looked at
    for (size_t i = 0; i < sizes.size(); ++i)
        if (sizes[i] > 1) left |= 1u << i;
    for (int64_t span = 1; left != 0;) {
        size_t low = 0;
        for (size_t i = 0, found = 0; i < sizes.size(); ++i)
            if ((left >> i & 1) != 0 && (found == 0 || strides[i] < strides[low])) { low = i; found = 1; }
        if (strides[low] < span) return true;
        span += (sizes[low] - 1) * strides[low];
        left &= ~(1u << low);
    }
    return false;
}

// A tensor that a call writes in place: autograd is told, so that a backward pass which saved what was there before is refused.
inline void check_written(const at::Tensor& t) {
    check(!(at::GradMode::is_enabled() && t.requires_grad()), "a tensor that requires a gradient cannot be written in place");
}
inline void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether two row tensors may share elements: false where their addresses do not meet, or where they are slices of one buffer
// side by side in every token (the queries and keys of one matrix product).
inline bool may_meet(const at::Tensor& a, const at::Tensor& b) {
    if (!Extent(a).meets(Extent(b))) return false;
    const char *pa = static_cast<const char*>(a.data_ptr()), *pb = static_cast<const char*>(b.data_ptr());
    const RowStrides sa = strides_of(a), sb = strides_of(b);
    const int64_t step = sa.s[1], size = a.element_size();
    if (step <= 0 || sb.s[1] != step || sa.s[0] % step != 0 || sb.s[0] % step != 0 || (pb - pa) % size != 0) return true;
    auto span = [](const at::Tensor& t) { return (t.size(-2) - 1) * t.stride(-2) + (t.size(-1) - 1) * t.stride(-1) + 1; };
    const int64_t apart = ((pb - pa) / size % step + step) % step;
    return span(a) > apart || apart + span(b) > step;
}
inline bool same_view(const at::Tensor& a, const at::Tensor& b) { return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides(); }

// What a result is written to: `out`, checked against all inputs, or new memory.
inline at::Tensor rows_out(const MaybeTensor& out, const at::Tensor& x, const at::Tensor& original, const MaybeTensor& other, const char* name) {
    if (!out.has_value()) return new_tensor(x.sizes(), x.scalar_type(), x);
    check_place(*out, x, name);
    check(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type(), "out must have the shape and dtype of its input");
    check(out->stride(-1) == 1 || out->size(-1) <= 1, "out must have contiguous rows");
    check(!rows_meet(*out), "rows of out must not share memory");
    check(same_view(*out, original) || !may_meet(*out, original), "out must be its input itself or share no memory with it");
    check(!other.has_value() || !may_meet(*out, *other), "out must share no memory with the other operands");
    check_written(*out);
    return *out;
}

struct Angles {
    at::Tensor positions, inv_freq;
    int bytes = 8, half = 0;
    int64_t batch_stride = 0;
};
inline Angles angles_of(const at::Tensor& positions, const at::Tensor& inv_freq, const at::Tensor& x) {
    check_place(positions, x, "positions");
    check_place(inv_freq, x, "inv_freq");
    check(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "positions must be int32 or int64");
    check(inv_freq.dim() == 1 && inv_freq.size(0) >= 1 && inv_freq.scalar_type() == at::kDouble, "inv_freq must be float64 of shape (rotary_dim / 2,)");
    check(2 * inv_freq.size(0) <= x.size(-1), "inv_freq has more pairs than a head");
    Angles a;
    const bool batched = x.dim() == 4;
    if (positions.dim() == 1) {
        check(positions.size(0) == x.size(batched ? 1 : 0), "positions must hold one value per token");
    } else {
        check(batched && positions.dim() == 2 && positions.size(0) == x.size(0) && positions.size(1) == x.size(1), "positions must have the shape of the tokens");
        a.batch_stride = positions.size(1);
    }
    a.positions = positions.contiguous();
    a.inv_freq = inv_freq.contiguous();
    a.bytes = positions.scalar_type() == at::kLong ? 8 : 4;
    a.half = int(inv_freq.size(0));
    return a;
}

struct Cache {
    int64_t s[3];
};
// Whether two caches may share rows: false where their addresses do not meet, or where both go on by one step, of blocks, tokens or heads,
// within which their rows lie side by side (the halves of one tensor, keys and values of a head in one row).
inline bool caches_may_meet(const at::Tensor& a, const at::Tensor& b) {
    if (!Extent(a).meets(Extent(b))) return false;
    const int64_t size = a.element_size();
    const int64_t between = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
    if (between % size != 0) return true;
    // the elements of t within one step, and whether all larger strides are whole steps
    auto within = [](const at::Tensor& t, int64_t step, int64_t& span) {
        span = 1;
        for (int64_t i = 0; i < t.dim(); ++i) {
            if (t.size(i) == 1) continue;
            if (t.stride(i) < step) span += (t.size(i) - 1) * t.stride(i);
            else if (t.stride(i) % step != 0) return false;
        }
        return true;
    };
    for (int64_t i = 0; i < a.dim(); ++i) {
        const int64_t step = a.stride(i);
        int64_t span_a, span_b;
        if (a.size(i) == 1 || step <= 0 || !within(a, step, span_a) || !within(b, step, span_b)) continue;
        const int64_t apart = (between / size % step + step) % step;
        if (span_a <= apart && apart + span_b <= step) return false;
    }
    return true;
}

inline Cache cache_of(const at::Tensor& cache, const at::Tensor& like, const at::Tensor& rows, const char* name) {
    check_place(cache, like, name);
    check(cache.dim() == 4 && cache.size(3) == rows.size(-1) && cache.scalar_type() == rows.scalar_type(),
          "key and value caches must have shape (num_blocks, block_size, H_KV, D) and the dtype of the rows");
    check(cache.stride(3) == 1 || cache.size(3) <= 1, "rows of the caches must be contiguous");
    return {{cache.stride(0), cache.stride(1), cache.stride(2)}};
}

}  // namespace
