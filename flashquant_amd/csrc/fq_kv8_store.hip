// The store into a paged cache of 8-bit rows, with rotary positions, and the way back.
//
//   y = rotary(x)  (keys; values: x),  E = the least power with max |y_i| <= 448 2^E,  code_i = e4m3(y_i 2^-E)
//
// for every row, the D values of a token and KV head; E goes beside the codes as an E8M0 byte (E + 127).  A power of two costs the
// codes nothing: their relative precision is the same in every binade, so a scale in between would gain at most part of one
// binade at the bottom of the range; products by it are exact, and a row's byte is 1/D of its codes where a float32 would be
// 4/D.  Keys are quantised from the float32 results of the rotation, not from these rounded to 16 bits.
//
// What bounds it: each row is read and written once, so HBM does; for the few tokens of a decode step the launch and one trip to
// memory do.  A row is 4, 8 or 16 neighbouring lanes of 16 values, the two eights of which lie apart as the pairs of a rotation do;
// its maximum takes two to four DPP moves.  Angles: one pair a thread, into LDS, for all heads of a token.
// Measured (whole calls): 48 tokens of 16 + 2 x 4 heads of 256 5.3 us; 9001 of 32 + 2 x 8 of 128 36 us, 203 MB, where a copy of as many bytes takes 39;
// back to 16 bits, three sequences of up to 700 tokens 5.2 us, 44,000 tokens of 8 heads (275 MB, two thirds of them written) 68 us, and 61
// into an output that is used again.
#include <type_traits>

#include "fq_kv8.hpp"
#include "fq_rotary.hpp"

namespace fq {

struct Store8Rows {
    const uint16_t* src;
    int64_t token;                              // strides in elements
    int head;
    int heads;
};

struct Store8Params {
    Store8Rows q, k, v;
    uint16_t* q_out;
    int64_t q_out_token;
    int q_out_head;
    const void* positions;
    int wide_positions;                         // int64, else int32
    const double* inv_freq;
    const int64_t* slots;
    uint8_t *key_codes, *value_codes, *key_scales, *value_scales;
    int64_t k_block, v_block, ks_block, vs_block;
    int k_token, k_head, v_token, v_head, ks_head, vs_head;
    int64_t num_slots, mapped, rows;            // rows: tokens times heads
    int page_log2, half, heads;                 // heads: of q, k and v together
    uint32_t heads_magic;
    float scale;
};

__device__ __forceinline__ int64_t position_of(const Store8Params& p, int64_t token) {
    return p.wide_positions ? static_cast<const int64_t*>(p.positions)[token] : int64_t(static_cast<const int32_t*>(p.positions)[token]);
}
// scale times cos and sin of a pair's angle, rounded once: the nearest quarter turn is taken off exactly, then the Taylor series,
// whose next terms are below 2^-36, all in 64 bits.  With both in 32 bits three times as many codes fell on the other side of a
// rounding; a thread has at most four pairs, which costs nothing that could be measured.
__device__ __forceinline__ float2v turn_of(const Store8Params& p, int64_t position, int pair) {
    const double x = double(position) * p.inv_freq[pair] * 0.15915494309189533576888;
    const double quarter = __builtin_rint(4.0 * x);
    const double t = __builtin_fma(-0.25, quarter, x) * 6.283185307179586476925287, z = t * t;
    double s = -1.0 / 39916800, c = 1.0 / 479001600;
    s = __builtin_fma(z, s, 1.0 / 362880);
    c = __builtin_fma(z, c, -1.0 / 3628800);
    s = __builtin_fma(z, s, -1.0 / 5040);
    c = __builtin_fma(z, c, 1.0 / 40320);
    s = __builtin_fma(z, s, 1.0 / 120);
    c = __builtin_fma(z, c, -1.0 / 720);
    s = __builtin_fma(z, s, -1.0 / 6);
    c = __builtin_fma(z, c, 1.0 / 24);
    s = __builtin_fma(t * z, s, t);
    c = __builtin_fma(z, __builtin_fma(z, c, -0.5), 1.0);
    const int k = int(quarter - 4.0 * __builtin_floor(0.25 * quarter));      // 0 .. 3
    const double a = (k & 1) ? s : c, b = (k & 1) ? c : s, scale = p.scale;
    return float2v{float(scale * (k == 1 || k == 2 ? -a : a)), float(scale * (k >= 2 ? -b : b))};
}

// The power of a row whose largest finite magnitude is `most`: 2^-8 of its binade, and one more where it lies above 1.75 of it
// (448 = 1.75 2^8).  A row of zeros has the lowest.
__device__ __forceinline__ int power_of(float most) {
    const uint32_t bits = float_to_bits(most);
    const int power = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return power < kRowPowerMin ? kRowPowerMin : power > kRowPowerMax ? kRowPowerMax : power;
}
__device__ __forceinline__ float finite_size(float y) {
    const float a = __builtin_fabsf(y);
    return a < __builtin_inff() ? a : 0.0f;                     // (NaN too)
}
// Four values as codes, to nearest even.  What is infinite becomes NaN, as e4m3 has no infinities.
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d, float down) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c * down, d * down, w, true));
}

// Row `row` of the launch: its token, and where it comes from and goes to.
struct Store8Place {
    int64_t token;
    int head;
    bool is_q, is_v, wanted;
    const uint16_t* src;
    uint8_t *codes, *scale;
};
__device__ __forceinline__ Store8Place place_of(const Store8Params& p, int64_t token, int h) {
    Store8Place r;
    r.token = token;
    r.is_q = h < p.q.heads;
    r.is_v = h >= p.q.heads + p.k.heads;
    if (!r.is_q) h -= p.q.heads;
    if (r.is_v) h -= p.k.heads;
    r.head = h;
    r.wanted = true;
    r.codes = r.scale = nullptr;
    r.src = r.is_q ? p.q.src + token * p.q.token + int64_t(h) * p.q.head
                   : r.is_v ? p.v.src + token * p.v.token + int64_t(h) * p.v.head : p.k.src + token * p.k.token + int64_t(h) * p.k.head;
    if (!r.is_q) {
        const int64_t slot = token < p.mapped ? p.slots[token] : -1;
        r.wanted = uint64_t(slot) < uint64_t(p.num_slots);
        if (r.wanted) {
            const int64_t block = slot >> p.page_log2;
            const int at = int(slot & ((1 << p.page_log2) - 1));
            r.codes = r.is_v ? p.value_codes + block * p.v_block + int64_t(at) * p.v_token + int64_t(h) * p.v_head
                             : p.key_codes + block * p.k_block + int64_t(at) * p.k_token + int64_t(h) * p.k_head;
            r.scale = r.is_v ? p.value_scales + block * p.vs_block + int64_t(h) * p.vs_head + at
                             : p.key_scales + block * p.ks_block + int64_t(h) * p.ks_head + at;
        }
    }
    return r;
}

constexpr int kStore8Threads = 256;
// angles of a workgroup's tokens: 16 rows of 256 coordinates reach into 8 tokens of two heads, 32 of 128 into 16, 64 of 64 into 32 (the
// first row of each is a token's first), and into 6, 12 and 22 of three
constexpr int kStore8Pairs = 1024;

template <int D, int DT, bool INTERLEAVED, bool STREAM>
__global__ __launch_bounds__(kStore8Threads) void rotary_store8_kernel(const Store8Params p) {
    constexpr int U = D / 16;                                  // lanes of a row
    constexpr int R = kStore8Threads / U;                      // rows of a workgroup
    __shared__ __align__(16) float2v turns[kStore8Pairs];
    const int64_t row0 = int64_t(blockIdx.x) * R;
    const int rows = int(p.rows - row0 < R ? p.rows - row0 : R);
    const int64_t token0 = row0 / p.heads;
    const uint32_t head0 = uint32_t(row0 - token0 * p.heads);
    const int row = int(threadIdx.x) / U, unit = int(threadIdx.x) % U;
    const int t = int(divide(row + head0, p.heads, p.heads_magic));
    Store8Place at;
    at.wanted = row < rows;
    if (at.wanted) at = place_of(p, token0 + t, int(row + head0) - t * p.heads);
    // the two eights of a piece lie apart: pairs of a rotation, or halves of what follows
    const int rotated = p.half / 8;
    const bool turned = at.wanted && !at.is_v && unit < rotated;
    const int rest0 = !at.wanted || at.is_v ? 0 : 2 * p.half, part = !at.wanted || at.is_v ? unit : unit - rotated;
    const int c0 = turned ? 8 * unit : rest0 + 8 * part, c1 = turned ? 8 * unit + p.half : c0 + (D - rest0) / 2;
    uint4v a = {0u, 0u, 0u, 0u}, d = a;
    if (at.wanted) {
        const uint4v *pa = reinterpret_cast<const uint4v*>(at.src + c0), *pd = reinterpret_cast<const uint4v*>(at.src + c1);
        a = STREAM ? __builtin_nontemporal_load(pa) : *pa;
        d = STREAM ? __builtin_nontemporal_load(pd) : *pd;
    }
    const int tokens = int((uint32_t(rows) + head0 - 1) / uint32_t(p.heads)) + 1;
    for (int i = threadIdx.x; i < tokens * p.half; i += kStore8Threads) {
        const int n = i / p.half;
        turns[i] = turn_of(p, position_of(p, token0 + n), i - n * p.half);
    }
    __syncthreads();
    float ya[8], yd[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ya[2 * i] = load_elem<DT>(uint16_t(a[i] & 0xffffu)); ya[2 * i + 1] = load_elem<DT>(uint16_t(a[i] >> 16));
        yd[2 * i] = load_elem<DT>(uint16_t(d[i] & 0xffffu)); yd[2 * i + 1] = load_elem<DT>(uint16_t(d[i] >> 16));
    }
    if (turned) {
        const float2v* cs = turns + t * p.half + (INTERLEAVED ? 4 : 8) * unit;
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2v y = turned_pair(ya[2 * i], ya[2 * i + 1], cs[i]), z = turned_pair(yd[2 * i], yd[2 * i + 1], cs[p.half / 2 + i]);
                ya[2 * i] = y.x; ya[2 * i + 1] = y.y;
                yd[2 * i] = z.x; yd[2 * i + 1] = z.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2v y = turned_pair(ya[i], yd[i], cs[i]);
                ya[i] = y.x;
                yd[i] = y.y;
            }
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fmaxf(finite_size(ya[i]), finite_size(yd[i])));
    // over the row's lanes
    most = __builtin_fmaxf(most, dpp_mov<0xb1>(most));                          // quad_perm 1 0 3 2
    most = __builtin_fmaxf(most, dpp_mov<0x4e>(most));                          // quad_perm 2 3 0 1
    if constexpr (U >= 8) most = __builtin_fmaxf(most, dpp_mov<0x141>(most));   // row_half_mirror
    if constexpr (U >= 16) most = __builtin_fmaxf(most, dpp_mov<0x140>(most));  // row_mirror
    if (!at.wanted) return;
    if (at.is_q) {
        uint16_t* dst = p.q_out + at.token * p.q_out_token + int64_t(at.head) * p.q_out_head;
        if (!turned && dst == at.src) return;                  // (what is rotated in place need not be copied)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = rounded_words<DT>(ya[2 * i], ya[2 * i + 1]);
            d[i] = rounded_words<DT>(yd[2 * i], yd[2 * i + 1]);
        }
        *reinterpret_cast<uint4v*>(dst + c0) = a;
        *reinterpret_cast<uint4v*>(dst + c1) = d;
        return;
    }
    const int power = power_of(most);
    const float down = bits_to_float(uint32_t(127 - power) << 23);
    *reinterpret_cast<uint2v*>(at.codes + c0) = uint2v{codes_of(ya[0], ya[1], ya[2], ya[3], down), codes_of(ya[4], ya[5], ya[6], ya[7], down)};
    *reinterpret_cast<uint2v*>(at.codes + c1) = uint2v{codes_of(yd[0], yd[1], yd[2], yd[3], down), codes_of(yd[4], yd[5], yd[6], yd[7], down)};
    if (unit == 0) *at.scale = uint8_t(power + 127);
}

// The same for rows that cannot be read 16 bytes at a time and rotations that are no multiple of 16 coordinates: a wavefront a row,
// neighbouring lanes neighbouring coordinates, each with the other of its pair read again and an angle of its own.
template <int D, int DT, bool INTERLEAVED>
__global__ __launch_bounds__(kStore8Threads) void rotary_store8_any_kernel(const Store8Params p) {
    constexpr int E = D / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t row = int64_t(blockIdx.x) * (kStore8Threads / kWave) + threadIdx.x / kWave;
    if (row >= p.rows) return;
    const int64_t token = row / p.heads;
    const Store8Place at = place_of(p, token, int(row - token * p.heads));
    if (!at.wanted) return;
    const int64_t position = at.is_v ? 0 : position_of(p, token);
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = lane + kWave * e;
        y[e] = load_elem<DT>(at.src[c]);
        if (!at.is_v && c < 2 * p.half) {
            const bool second = INTERLEAVED ? (c & 1) != 0 : c >= p.half;
            const int other = INTERLEAVED ? c ^ 1 : second ? c - p.half : c + p.half;
            const float x = load_elem<DT>(at.src[other]);
            const float2v turn = turn_of(p, position, INTERLEAVED ? c / 2 : second ? c - p.half : c);
            y[e] = second ? turned_pair(x, y[e], turn).y : turned_pair(y[e], x, turn).x;
        }
    }
    if (at.is_q) {
        asm volatile("" ::: "memory");                         // all of the row is read before any of it is written: out may be q
        uint16_t* dst = p.q_out + at.token * p.q_out_token + int64_t(at.head) * p.q_out_head;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float v = y[e];
            if constexpr (DT == FQ_F16) asm("" : "+v"(v));
            dst[lane + kWave * e] = store_elem<DT>(v);
        }
        return;
    }
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) most = __builtin_fmaxf(most, finite_size(y[e]));
    const int power = power_of(wave_max(most));
    const float down = bits_to_float(uint32_t(127 - power) << 23);
#pragma unroll
    for (int e = 0; e < E; ++e) at.codes[lane + kWave * e] = uint8_t(codes_of(y[e], 0.0f, 0.0f, 0.0f, down) & 0xffu);
    if (lane == 0) *at.scale = uint8_t(power + 127);
}

// Tokens back as 16-bit rows, code 2^E rounded to the type (bfloat16: exact but for its smallest numbers), finite what is beyond it.  Reads a byte and writes
// two, HBM-bound.  A thread has N pieces of 16 values, 256 pieces apart, and asks for all of them before it uses one; a piece is an
// eight of each half of a row, so that a store of neighbouring threads takes whole lines (16 values in one place: 67 us for 60).
// The sequence of a workgroup's first token is found by 64 lanes at a time, a later token's from there.
struct Read8Params {
    const uint8_t *codes[2], *scales[2];        // keys, values
    uint16_t* out[2];
    const int32_t *table, *cu, *starts;         // starts may be null: 0
    int64_t block[2], scale_block[2], table_row;
    int token[2], head[2], scale_head[2];
    int64_t tokens;
    int S, H, max_blocks, num_blocks, page_log2;
    int units;                                  // pieces of 16 values of a token, keys and values
    int fill;                                   // zeros behind the last token
};

// The last i of 0 .. n - 1 with cu[i] <= t (0 where there is none); cu is not decreasing.
__device__ __forceinline__ int last_upto(const int32_t* cu, int n, int64_t t, int lane) {
    int lo = 0;
    while (n > 1) {
        const int step = (n + kWave - 1) / kWave, i = lane * step;
        const uint64_t below = __ballot(i < n && cu[lo + (i < n ? i : 0)] <= t);
        const int k = below == 0 ? 0 : 63 - __builtin_clzll(below);
        lo += k * step;
        n = n - k * step < step ? n - k * step : step;
    }
    return lo;
}

template <int D, int DT, int N>
__global__ __launch_bounds__(256) void paged_kv8_read_kernel(const Read8Params p) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t first = int64_t(blockIdx.x) * (256 * N), token0 = first / p.units;
    const uint32_t skipped = uint32_t(first - token0 * p.units);
    int s = last_upto(p.cu, p.S + 1, token0, lane);
    int64_t begin = p.cu[s], next = s < p.S ? p.cu[s + 1] : INT64_MAX;
    int64_t token[N], entry[N], place[N];
    int side[N], head[N], c[N];
    bool inside[N];                                  // a sequence's token
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t at = skipped + 256 * k + threadIdx.x, step = at / uint32_t(p.units);
        int unit = int(at - step * uint32_t(p.units));
        side[k] = unit >= p.units / 2 ? 1 : 0;
        unit -= side[k] * (p.units / 2);
        head[k] = unit / (D / 16);
        c[k] = 8 * (unit % (D / 16));                          // an eight of each half of the row
        token[k] = token0 + step;
        while (s < p.S && next <= token[k]) {                  // (empty sequences have no token of their own)
            begin = next;
            ++s;
            next = s < p.S ? int64_t(p.cu[s + 1]) : INT64_MAX;
        }
        inside[k] = token[k] < p.tokens && s < p.S;
        place[k] = token[k] - begin;
        entry[k] = -1;
        if (inside[k]) {
            const bool ahead = place[k] < 0;
            if (p.starts != nullptr) place[k] += p.starts[s];
            const int64_t e = place[k] >> p.page_log2;
            if (!ahead && place[k] >= 0 && e < p.max_blocks) entry[k] = int64_t(s) * p.table_row + e;
        }
    }
    int block[N];
#pragma unroll
    for (int k = 0; k < N; ++k) block[k] = entry[k] >= 0 ? p.table[entry[k]] : -1;
    uint4v w[N];
    uint32_t scale[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        w[k] = uint4v{0u, 0u, 0u, 0u};
        scale[k] = 0;
        if (uint32_t(block[k]) < uint32_t(p.num_blocks)) {
            const int v = side[k], in_page = int(place[k] & ((1 << p.page_log2) - 1));
            const uint8_t* src = p.codes[v] + int64_t(block[k]) * p.block[v] + int64_t(in_page) * p.token[v] + int64_t(head[k]) * p.head[v] + c[k];
            const uint2v a = *reinterpret_cast<const uint2v*>(src), b = *reinterpret_cast<const uint2v*>(src + D / 2);
            w[k] = uint4v{a.x, a.y, b.x, b.y};
            scale[k] = p.scales[v][int64_t(block[k]) * p.scale_block[v] + int64_t(head[k]) * p.scale_head[v] + in_page];
        }
    }
    auto write = [&](auto ends) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (token[k] >= p.tokens || !(inside[k] || p.fill)) continue;
            const float up = row_scale<0>(scale[k]);
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2v x = codes_f32<false>(w[k][i]) * up, y = codes_f32<true>(w[k][i]) * up;
                if constexpr (decltype(ends)::value) {
                    x = float2v{held<DT>(x.x), held<DT>(x.y)};
                    y = float2v{held<DT>(y.x), held<DT>(y.y)};
                }
                o[2 * i] = rounded_words<DT>(x.x, x.y);
                o[2 * i + 1] = rounded_words<DT>(y.x, y.y);
            }
            uint16_t* dst = p.out[side[k]] + (token[k] * p.H + head[k]) * D + c[k];
            const uint4v lo = {o[0], o[1], o[2], o[3]}, hi = {o[4], o[5], o[6], o[7]};
            *reinterpret_cast<uint4v*>(dst) = lo;
            *reinterpret_cast<uint4v*>(dst + D / 2) = hi;
        }
    };
    // Rows that can hold what is beyond the type are few, and looked for (of every value, 41,000 tokens of 8 heads of 128 60 -> 66 us).
    uint32_t highest = scale[0];
#pragma unroll
    for (int k = 1; k < N; ++k) highest = highest > scale[k] ? highest : scale[k];
    if (__any(highest >= (DT == FQ_BF16 ? 127 + 120 : 127 + 8))) write(std::true_type{});
    else write(std::false_type{});
}

}  // namespace fq

namespace {

template <int D, int DT>
int launch_store8(const fq::Store8Params& p, bool wide, bool interleaved, hipStream_t s) {
    const int64_t each = wide ? fq::kStore8Threads * 16 / D : fq::kStore8Threads / fq::kWave, groups = (p.rows + each - 1) / each;
    if (groups > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    const unsigned n = unsigned(groups);
    // what is too much for the shared cache is read past it: 9001 tokens of 32 + 8 + 8 heads of 128 39.6 -> 35.8 us, 4000 17.8 -> 19.2
    const bool stream = p.rows * D * 4 > (int64_t(128) << 20);
    if (!wide) {
        if (interleaved) fq::rotary_store8_any_kernel<D, DT, true><<<n, fq::kStore8Threads, 0, s>>>(p);
        else fq::rotary_store8_any_kernel<D, DT, false><<<n, fq::kStore8Threads, 0, s>>>(p);
    } else if (interleaved) {
        if (stream) fq::rotary_store8_kernel<D, DT, true, true><<<n, fq::kStore8Threads, 0, s>>>(p);
        else fq::rotary_store8_kernel<D, DT, true, false><<<n, fq::kStore8Threads, 0, s>>>(p);
    } else {
        if (stream) fq::rotary_store8_kernel<D, DT, false, true><<<n, fq::kStore8Threads, 0, s>>>(p);
        else fq::rotary_store8_kernel<D, DT, false, false><<<n, fq::kStore8Threads, 0, s>>>(p);
    }
    return fq_host::check_launch();
}

template <int D, int DT>
int launch_read8_type(const fq::Read8Params& p, hipStream_t s) {
    // four pieces a thread where there is enough for the card: 13 sequences, 41,000 tokens of 8 heads of 128 60 us, 71 with one; 3 of
    // 1300 tokens 5.7 and 5.0 (stores past the shared cache 67 us)
    const int64_t pieces = p.tokens * p.units;
    const bool many = pieces >= int64_t(4 * 1024) * fq_host::device_cu_count();
    const int64_t each = many ? 1024 : 256, groups = (pieces + each - 1) / each;
    if (groups > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    if (many) fq::paged_kv8_read_kernel<D, DT, 4><<<unsigned(groups), 256, 0, s>>>(p);
    else fq::paged_kv8_read_kernel<D, DT, 1><<<unsigned(groups), 256, 0, s>>>(p);
    return fq_host::check_launch();
}
template <int D>
int launch_read8(const fq::Read8Params& p, int dtype, hipStream_t s) {
    return dtype == FQ_BF16 ? launch_read8_type<D, FQ_BF16>(p, s) : launch_read8_type<D, FQ_F16>(p, s);
}

}  // namespace

extern "C" int fq_rotary_paged_store8(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int H_Q,
                                      const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int H_KV,
                                      const void* positions, int position_bytes, const double* inv_freq, int half, int interleaved,
                                      float scale, const int64_t* slot_mapping, int64_t num_mapped, uint8_t* key_cache,
                                      const int64_t* key_strides, uint8_t* value_cache, const int64_t* value_strides, uint8_t* key_scales,
                                      const int64_t* key_scale_strides, uint8_t* value_scales, const int64_t* value_scale_strides,
                                      int block_size, int64_t num_blocks, int64_t tokens, int D, int dtype, void* stream) {
    const int bad = check_rotary(tokens, H_Q, H_KV, half, D, position_bytes);
    if (bad != FQ_OK) return bad;
    if (!fq_host::supported_dim(D)) return FQ_ERR_UNSUPPORTED_DIM;
    if (H_KV == 0 || num_mapped < 0 || num_mapped > tokens || num_blocks < 0 || num_blocks > 0x7fffffffLL || tokens > (int64_t(1) << 40))
        return FQ_ERR_BAD_SHAPE;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (tokens == 0) return FQ_OK;
    if (!positions || !inv_freq || (H_Q > 0 && (!q || !q_strides || !q_out || !q_out_strides)) || !k || !k_strides || !v || !v_strides)
        return FQ_ERR_NULL_POINTER;
    const bool stored = num_mapped > 0 && num_blocks > 0;
    if ((num_mapped > 0 && !slot_mapping) || (stored && (!key_cache || !key_strides || !value_cache || !value_strides || !key_scales ||
                                                         !key_scale_strides || !value_scales || !value_scale_strides)))
        return FQ_ERR_NULL_POINTER;
    if (!fits(k_strides + 1, 1) || !fits(v_strides + 1, 1) || (H_Q > 0 && (!fits(q_strides + 1, 1) || !fits(q_out_strides + 1, 1)))) return FQ_ERR_BAD_SHAPE;
    if (stored && (!fits(key_strides + 1, 2) || !fits(value_strides + 1, 2) || !fits(key_scale_strides + 1, 1) || !fits(value_scale_strides + 1, 1)))
        return FQ_ERR_BAD_SHAPE;
    fq::Store8Params p = {};
    bool wide = half % 8 == 0 && wide_rows(k, k_strides, 2, 8) && wide_rows(v, v_strides, 2, 8);
    if (H_Q > 0) {
        wide = wide && wide_rows(q, q_strides, 2, 8) && wide_rows(q_out, q_out_strides, 2, 8);
        p.q = {static_cast<const uint16_t*>(q), q_strides[0], int(q_strides[1]), H_Q};
        p.q_out = static_cast<uint16_t*>(q_out);
        p.q_out_token = q_out_strides[0];
        p.q_out_head = int(q_out_strides[1]);
    }
    p.k = {static_cast<const uint16_t*>(k), k_strides[0], int(k_strides[1]), H_KV};
    p.v = {static_cast<const uint16_t*>(v), v_strides[0], int(v_strides[1]), H_KV};
    if (stored) {
        wide = wide && wide_rows(key_cache, key_strides, 3, 8) && wide_rows(value_cache, value_strides, 3, 8);
        p.k_block = key_strides[0]; p.k_token = int(key_strides[1]); p.k_head = int(key_strides[2]);
        p.v_block = value_strides[0]; p.v_token = int(value_strides[1]); p.v_head = int(value_strides[2]);
        p.ks_block = key_scale_strides[0]; p.ks_head = int(key_scale_strides[1]);
        p.vs_block = value_scale_strides[0]; p.vs_head = int(value_scale_strides[1]);
    }
    p.key_codes = key_cache; p.value_codes = value_cache; p.key_scales = key_scales; p.value_scales = value_scales;
    p.positions = positions;
    p.wide_positions = position_bytes == 8;
    p.inv_freq = inv_freq;
    p.slots = slot_mapping;
    p.mapped = num_mapped;
    p.num_slots = num_blocks * block_size;
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.half = half; p.heads = H_Q + 2 * H_KV;
    p.rows = tokens * p.heads;
    p.heads_magic = magic_of(p.heads);
    p.scale = scale;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool inter = interleaved != 0;
    switch (D) {
        case 64: return dtype == FQ_BF16 ? launch_store8<64, FQ_BF16>(p, wide, inter, s) : launch_store8<64, FQ_F16>(p, wide, inter, s);
        case 128: return dtype == FQ_BF16 ? launch_store8<128, FQ_BF16>(p, wide, inter, s) : launch_store8<128, FQ_F16>(p, wide, inter, s);
        default: return dtype == FQ_BF16 ? launch_store8<256, FQ_BF16>(p, wide, inter, s) : launch_store8<256, FQ_F16>(p, wide, inter, s);
    }
}

extern "C" int fq_paged_kv8_read(const uint8_t* key_cache, const int64_t* key_strides, const uint8_t* value_cache, const int64_t* value_strides,
                                 const uint8_t* key_scales, const int64_t* key_scale_strides, const uint8_t* value_scales,
                                 const int64_t* value_scale_strides, const int32_t* block_table, int64_t block_table_stride,
                                 const int32_t* cu_seqlens, const int32_t* starts, void* keys, void* values, int fill, int num_seqs,
                                 int64_t num_tokens, int H_KV, int D, int block_size, int max_blocks_per_seq, int64_t num_blocks, int dtype,
                                 void* stream) {
    if (num_seqs < 0 || num_seqs > (1 << 30) || num_tokens < 0 || num_tokens > (int64_t(1) << 40) || H_KV <= 0 || H_KV > 4096 ||
        max_blocks_per_seq <= 0 || num_blocks < 0 || num_blocks > 0x7fffffffLL || block_table_stride < 0)
        return FQ_ERR_BAD_SHAPE;
    if (!fq_host::supported_dim(D)) return FQ_ERR_UNSUPPORTED_DIM;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (num_tokens == 0) return FQ_OK;
    if (!keys || !values || !cu_seqlens || (num_seqs > 0 && !block_table)) return FQ_ERR_NULL_POINTER;
    if (num_blocks > 0 && (!key_cache || !key_strides || !value_cache || !value_strides || !key_scales || !key_scale_strides || !value_scales ||
                           !value_scale_strides))
        return FQ_ERR_NULL_POINTER;
    if (!fq_host::aligned(keys, 16) || !fq_host::aligned(values, 16)) return FQ_ERR_MISALIGNED;
    fq::Read8Params p = {};
    if (num_blocks > 0) {
        if (!wide_rows(key_cache, key_strides, 3, 16) || !wide_rows(value_cache, value_strides, 3, 16)) return FQ_ERR_MISALIGNED;
        if (!fits(key_strides + 1, 2) || !fits(value_strides + 1, 2) || !fits(key_scale_strides + 1, 1) || !fits(value_scale_strides + 1, 1))
            return FQ_ERR_BAD_SHAPE;
        const int64_t *rows[2] = {key_strides, value_strides}, *scales[2] = {key_scale_strides, value_scale_strides};
        for (int i = 0; i < 2; ++i) {
            p.block[i] = rows[i][0]; p.token[i] = int(rows[i][1]); p.head[i] = int(rows[i][2]);
            p.scale_block[i] = scales[i][0]; p.scale_head[i] = int(scales[i][1]);
        }
    }
    p.codes[0] = key_cache; p.codes[1] = value_cache; p.scales[0] = key_scales; p.scales[1] = value_scales;
    p.out[0] = static_cast<uint16_t*>(keys); p.out[1] = static_cast<uint16_t*>(values);
    p.table = block_table; p.cu = cu_seqlens; p.starts = starts; p.table_row = block_table_stride;
    p.tokens = num_tokens;
    p.S = num_seqs; p.H = H_KV; p.max_blocks = max_blocks_per_seq; p.num_blocks = int(num_blocks);
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.units = 2 * H_KV * (D / 16);
    p.fill = fill;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_read8<64>(p, dtype, s);
        case 128: return launch_read8<128>(p, dtype, s);
        default: return launch_read8<256>(p, dtype, s);
    }
}
