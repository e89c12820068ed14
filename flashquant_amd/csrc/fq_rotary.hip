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
// Measured: 16384 tokens of 32 + 8 heads of 128, bf16, 54.4 us (6.2 TB/s; a copy 5.9); 3001 of 16 + 4 heads of 256, 64 of them
// turned, fp16, 11.7 us; with the store 12000 tokens of 32 + 8 + 8 49.6 us (5.9 TB/s); 32 tokens 3.1 us.
#include "fq_rotary.hpp"

namespace fq {

struct RotaryRows {
    const void* src;
    void* dst;                                  // null: keys and values that go to the cache
    int64_t src_batch, dst_batch;               // strides in elements
    int src_token, src_head, dst_token, dst_head;
    int heads;
};

struct RotaryParams {
    RotaryRows q, k, v;                         // v: with a store only (heads 0 otherwise)
    const void* positions;
    int64_t positions_batch;                    // positions between batches (0: one row of positions for all of them)
    const double* inv_freq;
    const int64_t* slots;                       // with a store
    uint16_t *key_cache, *value_cache;
    int k_block, k_token, k_head, v_block, v_token, v_head;
    int64_t num_slots, mapped;
    int64_t batch_tokens;                       // of one batch
    int64_t rows;                               // tokens of all batches times heads
    int batched;                                // more than one batch
    int page_log2;
    int wide_positions;                         // int64, else int32
    int half, D, heads;                         // heads: q, k and v together
    int units, rotated, tail;                   // of a row: pieces of 2 VEC elements, those of them that are turned, first element after them
    int tail_units, v_units;                    // pieces of what follows them, and of a value row
    int group_rows;                             // rows of a workgroup
    uint32_t units_magic, heads_magic;          // ceil(2^32 / .)
    float scale, sign;                          // sign -1: negative angles
};

// VEC elements as they lie in memory, and as float32
template <typename T, int VEC> struct Piece {
    T e[VEC];
};
template <int DT, typename T> __device__ __forceinline__ float to_float(T raw) {
    if constexpr (DT == FQ_F32) return raw;
    else return load_elem<DT>(raw);
}
template <int DT, typename T> __device__ __forceinline__ T from_float(float v) {
    if constexpr (DT == FQ_F32) {
        return v;
    } else {
        if constexpr (DT == FQ_F16) asm("" : "+v"(v));       // two roundings everywhere: no v_fma_mixlo_f16 here and there
        return store_elem<DT>(v);
    }
}
template <typename T, int VEC, bool STREAM> __device__ __forceinline__ Piece<T, VEC> load_piece(const T* src) {
    if constexpr (VEC * sizeof(T) == 16) {
        const uint4v* p = reinterpret_cast<const uint4v*>(src);
        return __builtin_bit_cast(Piece<T, VEC>, STREAM ? __builtin_nontemporal_load(p) : *p);
    } else {
        return Piece<T, VEC>{{src[0]}};
    }
}
template <typename T, int VEC, bool STREAM> __device__ __forceinline__ void store_piece(T* dst, const Piece<T, VEC>& v) {
    if constexpr (VEC * sizeof(T) == 16) {
        uint4v* p = reinterpret_cast<uint4v*>(dst);
        if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(uint4v, v), p);
        else *p = __builtin_bit_cast(uint4v, v);
    } else {
        dst[0] = v.e[0];
    }
}

// The eight pairs of two 16-byte parts of 16-bit values, a word at a time: words of `a` and `d` hold two elements of a part each.
// `first`, `later`: angles of pairs 0 to 3 and of pairs 4 to 7.
template <int DT, bool INTERLEAVED, typename P>
__device__ __forceinline__ void turn_words(const float2v* first, const float2v* later, P& pa, P& pd) {
    uint4v a = __builtin_bit_cast(uint4v, pa), d = __builtin_bit_cast(uint4v, pd);
    auto lo = [](uint32_t w) { return load_elem<DT>(uint16_t(w & 0xffffu)); };
    auto hi = [](uint32_t w) { return load_elem<DT>(uint16_t(w >> 16)); };
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2v y = turned_pair(lo(a[i]), hi(a[i]), first[i]), z = turned_pair(lo(d[i]), hi(d[i]), later[i]);
            a[i] = rounded_words<DT>(y.x, y.y);
            d[i] = rounded_words<DT>(z.x, z.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2v* cs = i < 2 ? first + 2 * i : later + 2 * (i - 2);
            const float2v y = turned_pair(lo(a[i]), lo(d[i]), cs[0]), z = turned_pair(hi(a[i]), hi(d[i]), cs[1]);
            a[i] = rounded_words<DT>(y.x, z.x);
            d[i] = rounded_words<DT>(y.y, z.y);
        }
    }
    pa = __builtin_bit_cast(P, a);
    pd = __builtin_bit_cast(P, d);
}

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 2048;      // cosines and sines of a workgroup

// A workgroup's rows (token by token, of each the heads of q, k and v) are cut into pieces of 2 VEC elements: VEC pairs, or that many
// elements to be copied.  A thread has one piece (of rows with more pieces than threads, several) and asks for it before it
// computes its share of the cosines and sines: one a thread and many workgroups a CU were faster than two or four pieces
// a thread (16384 tokens of 40 heads of 128, bf16: 55.9 us for 58.6 and 65, before the code for one piece was simplified).
template <int DT, typename T, int VEC, bool INTERLEAVED, bool STORE, bool STREAM>
__global__ __launch_bounds__(kRotaryThreads, 6) void rotary_kernel(const RotaryParams p) {
    constexpr bool kAdjacent = INTERLEAVED && VEC == 1;      // a piece is one pair, of two neighbours
    __shared__ __align__(16) float2v turns[kRotaryPairs];
    const int64_t row0 = int64_t(blockIdx.x) * p.group_rows;
    const int rows = int(p.rows - row0 < p.group_rows ? p.rows - row0 : p.group_rows);
    const int64_t token0 = row0 / p.heads;
    const uint32_t head0 = uint32_t(row0 - token0 * p.heads);
    // a row's units may be more than the threads: then they go round
    const int across = p.units < kRotaryThreads ? p.units : kRotaryThreads;
    const int row = int(divide(threadIdx.x, across, p.units_magic)), unit0 = int(threadIdx.x) - row * across;
    const int t = int(divide(row + head0, p.heads, p.heads_magic));
    int h = int(row + head0) - t * p.heads;
    const bool is_q = h < p.q.heads;
    const bool is_v = STORE && h >= p.q.heads + p.k.heads;
    if (!is_q) h -= p.q.heads;
    if (is_v) h -= p.k.heads;
    const int64_t token = token0 + t;
    bool wanted = row < rows;
    const T* src = nullptr;
    T* dst = nullptr;
    if (wanted) {
        int64_t in_batch = token, b = 0;
        if (p.batched) {
            b = token / p.batch_tokens;
            in_batch = token - b * p.batch_tokens;
        }
        src = static_cast<const T*>(is_q ? p.q.src : is_v ? p.v.src : p.k.src) + b * (is_q ? p.q.src_batch : p.k.src_batch) +
              in_batch * (is_q ? p.q.src_token : is_v ? p.v.src_token : p.k.src_token) +
              int64_t(h) * (is_q ? p.q.src_head : is_v ? p.v.src_head : p.k.src_head);
        if (STORE && !is_q) {
            const int64_t slot = token < p.mapped ? p.slots[token] : -1;
            wanted = uint64_t(slot) < uint64_t(p.num_slots);
            const int64_t block = slot >> p.page_log2, in_block = slot & ((1 << p.page_log2) - 1);
            if (wanted)
                dst = reinterpret_cast<T*>(is_v ? p.value_cache + block * p.v_block + in_block * p.v_token + int64_t(h) * p.v_head
                                                : p.key_cache + block * p.k_block + in_block * p.k_token + int64_t(h) * p.k_head);
        } else {
            dst = static_cast<T*>(is_q ? p.q.dst : p.k.dst) + b * (is_q ? p.q.dst_batch : p.k.dst_batch) +
                  in_batch * (is_q ? p.q.dst_token : p.k.dst_token) + int64_t(h) * (is_q ? p.q.dst_head : p.k.dst_head);
        }
    }
    bool first = true;
    for (int unit = unit0; unit < p.units; unit += across) {
        // the two parts of a piece lie apart, so that a load of neighbouring threads takes whole lines
        const bool turned = !is_v && unit < p.rotated;
        const int copied0 = is_v ? 0 : p.tail, part = is_v ? unit : unit - p.rotated, parts = is_v ? p.v_units : p.tail_units;
        const int c0 = turned ? (kAdjacent ? 2 * unit : VEC * unit) : copied0 + VEC * part;
        const int c1 = turned ? (kAdjacent ? 2 * unit + 1 : VEC * unit + p.half) : copied0 + VEC * (part + parts);
        // (what is rotated in place need not be copied)
        const bool mine = wanted && (turned || (part < parts && dst != src));
        const bool both = turned || c1 < p.D;
        Piece<T, VEC> a, d;
        if (mine) {
            a = load_piece<T, VEC, STREAM>(src + c0);
            if (both) d = load_piece<T, VEC, STREAM>(src + c1);
        }
        if (first) {
            const int tokens = int((uint32_t(rows) + head0 - 1) / uint32_t(p.heads)) + 1;
            for (int i = threadIdx.x; i < tokens * p.half; i += kRotaryThreads) {
                const int n = i / p.half, pair = i - n * p.half;
                int64_t at = token0 + n;
                if (p.batched) {
                    const int64_t b = at / p.batch_tokens;
                    at = b * p.positions_batch + (at - b * p.batch_tokens);
                }
                const int64_t position = p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
                const double angle = double(position) * p.inv_freq[pair];
                float2v cs = turn_cos_sin(angle * 0.15915494309189533576888);
                cs.x *= p.scale;
                cs.y *= p.scale * p.sign;
                turns[i] = cs;
            }
            __syncthreads();
            first = false;
        }
        if (!mine) continue;
        if (turned) {
            const float2v* cs = turns + t * p.half + (INTERLEAVED && !kAdjacent ? VEC / 2 : VEC) * unit;
            if constexpr (VEC == 8) {
                turn_words<DT, INTERLEAVED>(cs, cs + (INTERLEAVED ? p.half / 2 : 4), a, d);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    // pair e of the piece: element e of each part, or where neighbours are pairs, VEC / 2 of the first part and
                    // as many of the second, whose angles lie half of all further on
                    constexpr bool kInside = INTERLEAVED && !kAdjacent;
                    const bool later = kInside && 2 * e >= VEC;
                    T& lo = kInside ? (later ? d.e[(2 * e) % VEC] : a.e[(2 * e) % VEC]) : a.e[e];
                    T& hi = kInside ? (later ? d.e[(2 * e + 1) % VEC] : a.e[(2 * e + 1) % VEC]) : d.e[e];
                    const float2v turn = later ? cs[p.half / 2 + e - VEC / 2] : cs[e];
                    const float2v y = turned_pair(to_float<DT, T>(lo), to_float<DT, T>(hi), turn);
                    lo = from_float<DT, T>(y.x);
                    hi = from_float<DT, T>(y.y);
                }
            }
        }
        store_piece<T, VEC, STREAM>(dst + c0, a);
        if (both) store_piece<T, VEC, STREAM>(dst + c1, d);
    }
}

}  // namespace fq

namespace {

template <int DT, typename T, int VEC, bool STORE, bool STREAM>
void launch_rows(const fq::RotaryParams& p, bool interleaved, unsigned groups, hipStream_t s) {
    if (interleaved) fq::rotary_kernel<DT, T, VEC, true, STORE, STREAM><<<groups, fq::kRotaryThreads, 0, s>>>(p);
    else fq::rotary_kernel<DT, T, VEC, false, STORE, STREAM><<<groups, fq::kRotaryThreads, 0, s>>>(p);
}

template <int DT, typename T, bool STORE>
int launch_rotary(fq::RotaryParams& p, int64_t tokens, bool wide, bool interleaved, hipStream_t s) {
    constexpr int VEC = 16 / int(sizeof(T));
    const int vec = wide ? VEC : 1;
    p.rotated = p.half / vec;
    p.tail = 2 * p.half;
    const int rest = p.D - p.tail;
    p.tail_units = (rest + 2 * vec - 1) / (2 * vec);
    p.v_units = (p.D + 2 * vec - 1) / (2 * vec);
    p.units = p.rotated + p.tail_units;
    if (STORE && p.v_units > p.units) p.units = p.v_units;
    const int across = p.units < fq::kRotaryThreads ? p.units : fq::kRotaryThreads;
    p.rows = tokens * p.heads;
    // no more rows than there is room for the angles of the tokens that they reach into
    const int64_t most = int64_t(fq::kRotaryPairs / p.half - 1) * p.heads + 1;
    p.group_rows = fq::kRotaryThreads / across;
    if (p.group_rows > most) p.group_rows = int(most);
    p.units_magic = magic_of(across);
    p.heads_magic = magic_of(p.heads);
    const int64_t groups = (p.rows + p.group_rows - 1) / p.group_rows;
    if (groups > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    // What is too much for the 256 MB of shared cache, read and written, goes past it: copies of 168 MB took 58 us so and 63
    // otherwise, of 30 MB 11 and 9, and what is less is still there for whoever reads it next.
    const bool stream = p.rows * p.D * int64_t(2 * sizeof(T)) > (int64_t(256) << 20);
    const unsigned n = unsigned(groups);
    if (!wide) launch_rows<DT, T, 1, STORE, false>(p, interleaved, n, s);
    else if (stream) launch_rows<DT, T, VEC, STORE, true>(p, interleaved, n, s);
    else launch_rows<DT, T, VEC, STORE, false>(p, interleaved, n, s);
    return fq_host::check_launch();
}

fq::RotaryRows rows_of(const void* src, const int64_t* in, void* dst, const int64_t* out, int heads) {
    fq::RotaryRows r = {};
    r.src = src;
    r.dst = dst;
    r.src_batch = in[0]; r.src_token = int(in[1]); r.src_head = int(in[2]);
    if (out != nullptr) { r.dst_batch = out[0]; r.dst_token = int(out[1]); r.dst_head = int(out[2]); }
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
    for (const int64_t* st : {H_Q > 0 ? q_strides : nullptr, H_Q > 0 ? q_out_strides : nullptr, H_K > 0 ? k_strides : nullptr, H_K > 0 ? k_out_strides : nullptr})
        if (st != nullptr && !fits(st + 1, 2)) return FQ_ERR_BAD_SHAPE;
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
    p.batch_tokens = tokens;
    p.batched = batch > 1;
    p.half = half; p.D = D; p.heads = H_Q + H_K;
    p.scale = scale;
    p.sign = inverse ? -1.0f : 1.0f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case FQ_F16: return launch_rotary<FQ_F16, uint16_t, false>(p, batch * tokens, wide, interleaved != 0, s);
        case FQ_BF16: return launch_rotary<FQ_BF16, uint16_t, false>(p, batch * tokens, wide, interleaved != 0, s);
        default: return launch_rotary<FQ_F32, float, false>(p, batch * tokens, wide, interleaved != 0, s);
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
    if (!fits(k_strides, 2) || !fits(v_strides, 2) || (H_Q > 0 && (!fits(q_strides, 2) || !fits(q_out_strides, 2)))) return FQ_ERR_BAD_SHAPE;
    if (num_mapped > 0 && (!fits(key_strides, 3) || !fits(value_strides, 3))) return FQ_ERR_BAD_SHAPE;
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
        p.k_block = int(key_strides[0]); p.k_token = int(key_strides[1]); p.k_head = int(key_strides[2]);
        p.v_block = int(value_strides[0]); p.v_token = int(value_strides[1]); p.v_head = int(value_strides[2]);
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
    p.batch_tokens = tokens;
    p.half = half; p.D = D; p.heads = H_Q + 2 * H_KV;
    p.scale = scale;
    p.sign = 1.0f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == FQ_BF16 ? launch_rotary<FQ_BF16, uint16_t, true>(p, tokens, wide, interleaved != 0, s)
                            : launch_rotary<FQ_F16, uint16_t, true>(p, tokens, wide, interleaved != 0, s);
}
