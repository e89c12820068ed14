// Rotary positions on queries and keys, alone or with the store of keys and values into a 16-bit paged cache.
//
//   theta = position * inv_freq[i],  (y0, y1) = scale (x0 cos theta - x1 sin theta, x1 cos theta + x0 sin theta)
//
// for the pairs i of a head's first 2 * half coordinates: (i, i + half), or (2 i, 2 i + 1) where they are interleaved.  The
// rest of the head is copied.  The gradient, and the way back, is the same with -theta.
//
// What bounds it: each row is read and written once and a pair takes four multiply-adds, so HBM does; for the few tokens of a
// decode step the launch and one trip to memory do.  The angles are not read from a table (for 131,072 positions of 64 pairs 64
// MB, and 512 bytes a token): a workgroup computes the cosines and sines of its tokens, one pair a thread, into LDS, and all heads
// of these tokens use them.  The product and its reduction are in 64 bits: in 32 an angle at position 10^6 is off by 0.03.
#include "fq_device.hpp"

namespace fq {

struct RotaryRows {
    const void* src;
    void* dst;                                  // null: keys and values that go to the cache
    int64_t src_batch, src_token, src_head;     // strides in elements
    int64_t dst_batch, dst_token, dst_head;
    int heads;
};

struct RotaryParams {
    RotaryRows q, k, v;                         // v: with a store only (heads 0 otherwise)
    const void* positions;
    int64_t positions_batch;                    // positions between batches (0: one row of positions for all of them)
    const double* inv_freq;
    const int64_t* slots;                       // with a store
    uint16_t *key_cache, *value_cache;
    int64_t k_block, k_token, k_head, v_block, v_token, v_head;
    int64_t num_slots, mapped;
    int64_t tokens;                             // of all batches
    int64_t batch_tokens;                       // of one
    int page_log2;
    int wide_positions;                         // int64, else int32
    int half, D, heads;                         // heads: q, k and v together
    int units, rotated, tail;                   // of a row: pieces of 2 VEC elements, those of them that are turned, first after them
    int per_group;                              // tokens of a workgroup
    int rows_per_group;                         // (token, head) rows of a workgroup: per_group * heads, or a part of one token's heads
    int groups_per_token;
    uint32_t units_magic, heads_magic;          // ceil(2^32 / .)
    float scale;                                // negative angles: `sign` -1
    float sign;
};

// i / d for i d < 2^32, with magic = ceil(2^32 / d)
__device__ __forceinline__ uint32_t divide(uint32_t i, uint32_t d, uint32_t magic) { return d == 1 ? i : __umulhi(i, magic); }

// cos and sin of 2 pi x: the nearest quarter turn is taken off exactly, the rest, at most an eighth of a turn, goes through the
// Taylor series (next terms below 2^-40), in 64 bits throughout; one rounding at the end.
__device__ __forceinline__ float2v turn_cos_sin(double x) {
    const double quarter = __builtin_rint(4.0 * x);
    const double t = (x - 0.25 * quarter) * 6.283185307179586476925287;
    const double z = t * t;
    const double s = t * (1.0 + z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 - z * (1.0 / 39916800))))));
    const double c = 1.0 + z * (-1.0 / 2 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 + z * (-1.0 / 3628800 + z * (1.0 / 479001600))))));
    const int k = int(quarter - 4.0 * __builtin_floor(0.25 * quarter));      // 0 .. 3
    const double a = (k & 1) ? s : c, b = (k & 1) ? c : s;
    return float2v{float(k == 1 || k == 2 ? -a : a), float(k >= 2 ? -b : b)};
}

// VEC elements as they lie in memory, and as float32
template <typename T, int VEC> struct Piece {
    T e[VEC];
};
template <int DT, typename T> __device__ __forceinline__ float to_float(T raw) {
    if constexpr (DT == FQ_F32) return raw;
    else return load_elem<DT>(raw);
}
template <int DT, typename T> __device__ __forceinline__ T from_float(float v) {
    if constexpr (DT == FQ_F32) return v;
    else return store_elem<DT>(v);
}
template <typename T, int VEC> __device__ __forceinline__ Piece<T, VEC> load_piece(const T* src) {
    if constexpr (VEC * sizeof(T) == 16) return __builtin_bit_cast(Piece<T, VEC>, *reinterpret_cast<const uint4v*>(src));
    else return Piece<T, VEC>{{src[0]}};
}
template <typename T, int VEC> __device__ __forceinline__ void store_piece(T* dst, const Piece<T, VEC>& v) {
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4v*>(dst) = __builtin_bit_cast(uint4v, v);
    else dst[0] = v.e[0];
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 1024;      // cosines and sines of a workgroup

template <int DT, typename T, int VEC, bool INTERLEAVED, bool STORE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryParams p) {
    __shared__ __align__(16) float2v turns[kRotaryPairs];
    const int64_t group = blockIdx.x / p.groups_per_token;
    const int piece_of_token = int(blockIdx.x - group * p.groups_per_token);
    const int64_t first = group * p.per_group;
    const int tokens = int(p.tokens - first < p.per_group ? p.tokens - first : p.per_group);
    for (int i = threadIdx.x; i < tokens * p.half; i += kRotaryThreads) {
        const int t = i / p.half, pair = i - t * p.half;
        const int64_t token = first + t;
        int64_t at = token;
        if (p.batch_tokens != p.tokens) {
            const int64_t b = token / p.batch_tokens;
            at = b * p.positions_batch + (token - b * p.batch_tokens);
        }
        const int64_t position = p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
        const double angle = double(position) * p.inv_freq[pair];
        float2v cs = turn_cos_sin(angle * 0.15915494309189533576888);
        cs.x *= p.scale;
        cs.y *= p.scale * p.sign;
        turns[i] = cs;
    }
    __syncthreads();
    // rows of the workgroup: token by token, of each q, k and v heads
    const int row0 = piece_of_token * p.rows_per_group;
    const int rows = p.groups_per_token > 1 ? (p.heads - row0 < p.rows_per_group ? p.heads - row0 : p.rows_per_group) : tokens * p.heads;
    for (uint32_t i = threadIdx.x; i < uint32_t(rows) * uint32_t(p.units); i += kRotaryThreads) {
        const uint32_t r = divide(i, p.units, p.units_magic);
        const int unit = int(i - r * p.units);
        const uint32_t t = divide(r + row0, p.heads, p.heads_magic);
        int h = int(r + row0 - t * p.heads);
        const int64_t token = first + t;
        const bool is_q = h < p.q.heads;
        const bool is_v = STORE && h >= p.q.heads + p.k.heads;
        if (!is_q) h -= p.q.heads;
        if (is_v) h -= p.k.heads;
        const RotaryRows& x = is_q ? p.q : is_v ? p.v : p.k;
        int64_t b = 0, in_batch = token;
        if (p.batch_tokens != p.tokens) {
            b = token / p.batch_tokens;
            in_batch = token - b * p.batch_tokens;
        }
        const T* src = static_cast<const T*>(x.src) + b * x.src_batch + in_batch * x.src_token + h * x.src_head;
        T* dst;
        if (STORE && !is_q) {
            if (token >= p.mapped) continue;
            const int64_t slot = p.slots[token];
            if (uint64_t(slot) >= uint64_t(p.num_slots)) continue;
            const int64_t block = slot >> p.page_log2, in_block = slot & ((1 << p.page_log2) - 1);
            dst = reinterpret_cast<T*>(is_v ? p.value_cache + block * p.v_block + in_block * p.v_token + h * p.v_head
                                            : p.key_cache + block * p.k_block + in_block * p.k_token + h * p.k_head);
        } else {
            dst = static_cast<T*>(x.dst) + b * x.dst_batch + in_batch * x.dst_token + h * x.dst_head;
        }
        const bool turned = !is_v && unit < p.rotated;
        int c0, c1;
        if (turned) {
            c0 = INTERLEAVED ? 2 * VEC * unit : VEC * unit;
            c1 = INTERLEAVED ? c0 + VEC : c0 + p.half;
        } else {
            c0 = is_v ? 2 * VEC * unit : p.tail + 2 * VEC * (unit - p.rotated);
            c1 = c0 + VEC;
            if (c0 >= p.D || dst == src) continue;
        }
        const bool second = turned || c1 < p.D;
        Piece<T, VEC> a = load_piece<T, VEC>(src + c0), d = a;
        if (second) d = load_piece<T, VEC>(src + c1);
        if (turned) {
            const float2v* cs = turns + t * p.half + VEC * unit;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                // pair e of the piece: elements 2 e and 2 e + 1 of the two halves together, or e of each
                T& lo = INTERLEAVED ? (2 * e < VEC ? a.e[(2 * e) % VEC] : d.e[(2 * e) % VEC]) : a.e[e];
                T& hi = INTERLEAVED ? (2 * e + 1 < VEC ? a.e[(2 * e + 1) % VEC] : d.e[(2 * e + 1) % VEC]) : d.e[e];
                const float x0 = to_float<DT, T>(lo), x1 = to_float<DT, T>(hi), c = cs[e].x, s = cs[e].y;
                // (which product is rounded is spelled out: the same bits at every alignment)
                lo = from_float<DT, T>(__builtin_fmaf(x0, c, -(x1 * s)));
                hi = from_float<DT, T>(__builtin_fmaf(x1, c, x0 * s));
            }
        }
        store_piece<T, VEC>(dst + c0, a);
        if (second) store_piece<T, VEC>(dst + c1, d);
    }
}

}  // namespace fq

namespace {

uint32_t magic_of(int d) { return uint32_t(((uint64_t(1) << 32) + uint32_t(d) - 1) / uint32_t(d)); }

// whether rows at `ptr` with these strides can be read and written 16 bytes at a time
bool wide_rows(const void* ptr, const int64_t* strides, int n, int vec) {
    if (!fq_host::aligned(ptr, 16)) return false;
    for (int i = 0; i < n; ++i)
        if (strides[i] % vec != 0) return false;
    return true;
}

template <int DT, typename T, bool STORE>
int launch_rotary(fq::RotaryParams& p, bool wide, bool interleaved, hipStream_t s) {
    constexpr int VEC = 16 / int(sizeof(T));
    const int vec = wide ? VEC : 1;
    p.rotated = p.half / vec;
    p.tail = 2 * p.half;
    const int rest = p.D - p.tail;
    p.units = p.rotated + (rest + 2 * vec - 1) / (2 * vec);
    if (STORE && (p.D + 2 * vec - 1) / (2 * vec) > p.units) p.units = (p.D + 2 * vec - 1) / (2 * vec);
    // A workgroup's rows are as many tokens' as give every thread about five pieces, so that its cosines and sines serve all heads;
    // where the tokens are too few to fill the card so, one token's heads are spread over several workgroups, a piece a thread.
    const int64_t per_token = int64_t(p.heads) * p.units;
    int64_t tokens = (5 * fq::kRotaryThreads + per_token - 1) / per_token;
    const int64_t most = fq::kRotaryPairs / p.half;
    const int64_t fill = p.tokens / (2 * fq_host::device_cu_count());
    tokens = tokens > fill ? fill : tokens;
    tokens = tokens > most ? most : tokens;
    tokens = tokens < 1 ? 1 : tokens;
    p.per_group = int(tokens);
    p.groups_per_token = 1;
    p.rows_per_group = int(tokens) * p.heads;
    if (tokens == 1) {
        const int rows = p.units >= fq::kRotaryThreads ? 1 : fq::kRotaryThreads / p.units;
        const int64_t spread = (p.heads + rows - 1) / rows;
        if (spread > 1 && p.tokens * spread <= 8 * int64_t(fq_host::device_cu_count())) {
            p.groups_per_token = int(spread);
            p.rows_per_group = rows;
        }
    }
    p.units_magic = magic_of(p.units);
    p.heads_magic = magic_of(p.heads);
    const int64_t groups = (p.tokens + tokens - 1) / tokens * p.groups_per_token;
    if (groups > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    const dim3 grid(static_cast<unsigned>(groups)), block(fq::kRotaryThreads);
    if (wide && interleaved) fq::rotary_kernel<DT, T, VEC, true, STORE><<<grid, block, 0, s>>>(p);
    else if (wide) fq::rotary_kernel<DT, T, VEC, false, STORE><<<grid, block, 0, s>>>(p);
    else if (interleaved) fq::rotary_kernel<DT, T, 1, true, STORE><<<grid, block, 0, s>>>(p);
    else fq::rotary_kernel<DT, T, 1, false, STORE><<<grid, block, 0, s>>>(p);
    return fq_host::check_launch();
}

int check_rotary(int64_t tokens, int H_Q, int H_K, int half, int D, int position_bytes) {
    if (tokens < 0 || H_Q < 0 || H_K < 0 || H_Q + int64_t(H_K) == 0 || H_Q > 4096 || H_K > 4096) return FQ_ERR_BAD_SHAPE;
    if (half < 1 || D < 2 * half || D > 1024) return FQ_ERR_BAD_SHAPE;
    if (position_bytes != 4 && position_bytes != 8) return FQ_ERR_UNSUPPORTED_DTYPE;
    return FQ_OK;
}

fq::RotaryRows rows_of(const void* src, const int64_t* in, void* dst, const int64_t* out, int heads) {
    fq::RotaryRows r = {};
    r.src = src;
    r.dst = dst;
    r.src_batch = in[0]; r.src_token = in[1]; r.src_head = in[2];
    if (out != nullptr) { r.dst_batch = out[0]; r.dst_token = out[1]; r.dst_head = out[2]; }
    r.heads = heads;
    return r;
}

}  // namespace

extern "C" int fq_rotary_embedding(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int H_Q,
                                   const void* k, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides, int H_K,
                                   const void* positions, int position_bytes, int64_t positions_batch_stride, const double* inv_freq,
                                   int half, int interleaved, float scale, int inverse, int64_t batch, int64_t tokens, int D, int dtype,
                                   void* stream) {
    if (batch < 0) return FQ_ERR_BAD_SHAPE;
    const int bad = check_rotary(tokens, H_Q, H_K, half, D, position_bytes);
    if (bad != FQ_OK) return bad;
    if (dtype != FQ_F16 && dtype != FQ_BF16 && dtype != FQ_F32) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (batch == 0 || tokens == 0) return FQ_OK;
    if (tokens > (int64_t(1) << 40) / batch) return FQ_ERR_BAD_SHAPE;
    if (!positions || !inv_freq || (H_Q > 0 && (!q || !q_strides || !q_out || !q_out_strides)) ||
        (H_K > 0 && (!k || !k_strides || !k_out || !k_out_strides)))
        return FQ_ERR_NULL_POINTER;
    const int vec = dtype == FQ_F32 ? 4 : 8;
    bool wide = half % vec == 0 && D % vec == 0;
    fq::RotaryParams p = {};
    if (H_Q > 0) {
        p.q = rows_of(q, q_strides, q_out, q_out_strides, H_Q);
        wide = wide && wide_rows(q, q_strides, 3, vec) && wide_rows(q_out, q_out_strides, 3, vec);
    }
    if (H_K > 0) {
        p.k = rows_of(k, k_strides, k_out, k_out_strides, H_K);
        wide = wide && wide_rows(k, k_strides, 3, vec) && wide_rows(k_out, k_out_strides, 3, vec);
    }
    p.positions = positions;
    p.positions_batch = positions_batch_stride;
    p.wide_positions = position_bytes == 8;
    p.inv_freq = inv_freq;
    p.tokens = batch * tokens;
    p.batch_tokens = tokens;
    p.half = half; p.D = D; p.heads = H_Q + H_K;
    p.scale = scale;
    p.sign = inverse ? -1.0f : 1.0f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case FQ_F16: return launch_rotary<FQ_F16, uint16_t, false>(p, wide, interleaved != 0, s);
        case FQ_BF16: return launch_rotary<FQ_BF16, uint16_t, false>(p, wide, interleaved != 0, s);
        default: return launch_rotary<FQ_F32, float, false>(p, wide, interleaved != 0, s);
    }
}

extern "C" int fq_rotary_paged_store(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int H_Q,
                                     const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int H_KV,
                                     const void* positions, int position_bytes, const double* inv_freq, int half, int interleaved,
                                     float scale, const int64_t* slot_mapping, int64_t num_mapped, void* key_cache,
                                     const int64_t* key_strides, void* value_cache, const int64_t* value_strides, int block_size,
                                     int64_t num_blocks, int64_t tokens, int D, int dtype, void* stream) {
    const int bad = check_rotary(tokens, H_Q, H_KV, half, D, position_bytes);
    if (bad != FQ_OK) return bad;
    if (H_KV == 0 || num_mapped < 0 || num_mapped > tokens || num_blocks < 0 || num_blocks > 0x7fffffffLL || tokens > (int64_t(1) << 40))
        return FQ_ERR_BAD_SHAPE;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (tokens == 0) return FQ_OK;
    if (!positions || !inv_freq || (H_Q > 0 && (!q || !q_strides || !q_out || !q_out_strides)) || !k || !k_strides || !v || !v_strides)
        return FQ_ERR_NULL_POINTER;
    if (num_mapped > 0 && (!slot_mapping || (num_blocks > 0 && (!key_cache || !value_cache)) || !key_strides || !value_strides))
        return FQ_ERR_NULL_POINTER;
    bool wide = half % 8 == 0 && D % 8 == 0;
    fq::RotaryParams p = {};
    // one batch: the first stride is not looked at
    auto rows = [&](const void* src, const int64_t* in, void* dst, const int64_t* out, int heads) {
        const int64_t a[3] = {0, in[0], in[1]}, b[3] = {0, out ? out[0] : 0, out ? out[1] : 0};
        wide = wide && wide_rows(src, a, 3, 8) && (dst == nullptr || wide_rows(dst, b, 3, 8));
        return rows_of(src, a, dst, out ? b : nullptr, heads);
    };
    if (H_Q > 0) p.q = rows(q, q_strides, q_out, q_out_strides, H_Q);
    p.k = rows(k, k_strides, nullptr, nullptr, H_KV);
    p.v = rows(v, v_strides, nullptr, nullptr, H_KV);
    if (num_mapped > 0 && num_blocks > 0) {
        wide = wide && wide_rows(key_cache, key_strides, 3, 8) && wide_rows(value_cache, value_strides, 3, 8);
        p.k_block = key_strides[0]; p.k_token = key_strides[1]; p.k_head = key_strides[2];
        p.v_block = value_strides[0]; p.v_token = value_strides[1]; p.v_head = value_strides[2];
    }
    p.key_cache = static_cast<uint16_t*>(key_cache);
    p.value_cache = static_cast<uint16_t*>(value_cache);
    p.slots = slot_mapping;
    p.mapped = num_mapped;
    p.num_slots = num_blocks * block_size;
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.positions = positions;
    p.wide_positions = position_bytes == 8;
    p.inv_freq = inv_freq;
    p.tokens = p.batch_tokens = tokens;
    p.half = half; p.D = D; p.heads = H_Q + 2 * H_KV;
    p.scale = scale;
    p.sign = 1.0f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == FQ_BF16 ? launch_rotary<FQ_BF16, uint16_t, true>(p, wide, interleaved != 0, s)
                            : launch_rotary<FQ_F16, uint16_t, true>(p, wide, interleaved != 0, s);
}
