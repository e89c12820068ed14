// Attention of one new token per sequence over a paged cache of 16-bit keys and values.
//
//   o_h = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q_h . k_j - m),  c = sm_scale log2(e),  m = max_j c q_h . k_j
//
// over the tokens j of the sequence (with a window: the last ones); the G = H_Q / H_KV query heads of a KV head share its rows.
//
// What bounds it: every key and value is read once, 4 D bytes a token and KV head for 4 G D flops, so HBM does.  The tile loop
// therefore only has to keep enough loads in flight, and is laid out so that nothing but registers stands between a load and
// the matrix cores:
//   * A wavefront takes 32 keys at a time.  S^T = K Q^T and O^T = V^T P run on v_mfma_f32_16x16x32, heads along the columns.  Row m
//     of tile t of the scores is key 8 (m / 4) + 4 t + m % 4, so that after two tiles lane (g, h) holds the scores of keys 8 g ..
//     8 g + 7 for head h: exactly the B operand of the second product, without a move between lanes.  Maximum, sum and
//     rescaling of a head are a lane's own.
//   * A load takes whole lines of 128 bytes.  Of a key that is 64 coordinates, twice what the A operand holds: rows 0 to 7 of
//     the operand are eight keys' first halves, rows 8 to 15 their second halves; it is multiplied with both halves of the
//     query, and the right quarters of the two results are added across the halves of the wavefront.  That doubles a product that
//     costs nothing, where 64 bytes a key and load read every line twice (32 x 4096 tokens, 8 heads of 128, non-temporal: 105 us
//     for 95).
//   * A lane loads coordinates 8 n .. 8 n + 7 of the values of keys 8 g .. 8 g + 7 (whole rows) and turns them into the A operand, 8
//     keys of one coordinate, with half a v_perm_b32 an element; a key that is not seen becomes zero there, whatever it holds.
//   * Loads are non-temporal: a layer's keys and values are read once a step, and other layers' pass through the 256 MB of
//     shared cache in between (32 x 4096: 105 us -> 95; a stream of 2 GB of its own: 6.2 TB/s -> 7.0).
//   * The wavefronts of a workgroup take up to four neighbouring heads of the same tokens, whose rows lie side by side (against one
//     head a workgroup: 61 sequences of 500 to 16000 tokens, 64 heads over 8, 364 us -> 348; a plain read of the rows 6.6 ->
//     6.95 TB/s), and the tiles in turn; wavefronts of the same head are joined in LDS.
//   * A weight goes to the second product as two 16-bit terms (16 significant bits and more), so that the only rounding
//     that shows is that of the output; the matrix cores are idle otherwise.  Maximum and sum are float32, of the unrounded
//     weights.
// Measured: 32 sequences of 4096 tokens, 32 heads over 8 of 128, bf16, 84 us (6.4 TB/s); 61 of 500 to 16000, 64 over 8, fp16, 343 us
// (6.6 TB/s); 3 of 40000 to 65536, 8 heads over 1, 21 us; one of 777, 32 over 8, 9.2 us.
#include <type_traits>

#include "fq_device.hpp"

namespace fq {

constexpr int kKvTile = 32;               // keys of a wavefront's step
// Weights are kept times 2^lift.  fp16: up, so that their second terms stay normal.  bf16 has the exponents of float32, and a value may
// lie near 2^128: down, so that no wavefront's sum of up to 2^20 such values overflows where their average does not (what underflows
// instead are products below 2^-106).
template <int DT> constexpr float kKvLift = DT == FQ_F16 ? 10.0f : -20.0f;

struct KvDecodeParams {
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int32_t* table;
    const int32_t* lens;
    uint16_t* out;
    float* lse;                           // may be null
    float* part_o;                        // (S + shares, H_KV, G, D)
    float* part_m;                        // (S + shares, H_KV, G)
    float* part_l;
    int2* place;                          // (S): the share that holds a sequence's first tile, and the shares that hold tiles of it
    int64_t q_seq, q_head;                // strides in elements
    int64_t k_block, k_token, k_head, v_block, v_token, v_head;
    int64_t table_row;
    int S, H_KV, G, page_log2, max_blocks, num_blocks, window;
    int shares;                           // workgroups among which the tiles of a KV head are divided; 0: one a sequence
    int min_tiles;                        // of such a share
    float scale_log2;
};

// The tokens [lo, len) that sequence s sees, and the tiles that hold them.
struct KvSpan {
    int lo, len, first, tiles;
};
__device__ __forceinline__ KvSpan kv_span(const KvDecodeParams& p, int len) {
    KvSpan r;
    const int64_t room = int64_t(p.max_blocks) << p.page_log2;
    r.len = len < 0 ? 0 : len > room ? int(room) : len;
    r.lo = p.window > 0 && r.len > p.window ? r.len - p.window : 0;
    r.first = r.lo / kKvTile;
    r.tiles = (r.len + kKvTile - 1) / kKvTile - r.first;
    return r;
}

// How the work is divided where contexts may be long: the tiles of all sequences are cut into equal shares, one a workgroup (of a KV
// head), so that all of them end together whatever the lengths are.  Nothing on the host knows the lengths: every workgroup
// adds them up for itself.  Where there are shares enough, each belongs to one sequence, whose last one may be smaller (8 x 2000
// tokens, 32 heads over 8 of 128: 20.4 -> 17.9 us; 3 of 40000 to 65536, 8 over 1: 23.0 -> 21.4); otherwise the sequences are laid
// one after another before they are cut, and a share goes on from one to the next.  The piece of sequence s in share x is
// number x + s of the partial results: from one piece to the next either the share or the sequence goes up by one.
struct KvPlace {
    int size;                             // tiles of a share
    int seq, offset, left;                // the sequence where a share begins, its first tile there, the tiles of the share
    KvSpan span;
};
__device__ __forceinline__ int kv_len_of(const KvDecodeParams& p, int s) { return s < p.S ? p.lens[s] : 0; }

// The sum over this lane and those before it (a wavefront's length in six vector instructions).
__device__ __forceinline__ int sum_upto(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // row_bcast:31 into rows 2 and 3
    return v;
}

// Where share x begins.  False: there is no such share.  The lengths are read kGroups x 64 at a time, all of them asked for before
// the first is used, and up to that many only once (4096 sequences of 100 to 1200 tokens in a table for 4096, 8 heads over 1: 266 us,
// and 468 with 64 at a time here and in the second kernel; 1 x 777 tokens 9.2, and 9.4 with 512).
template <int kGroups>
__device__ __forceinline__ bool kv_place(const KvDecodeParams& p, int x, int lane, KvPlace& r) {
    constexpr int kAll = kGroups * kWave;
    int len[kGroups];
    auto read = [&](int s0) {
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            len[k] = 0;
            if (s0 + k * kWave < p.S) len[k] = kv_len_of(p, s0 + k * kWave + lane);
        }
    };
    // the sum of f(tiles) over the sequences, or over those that have been read
    auto sum_read = [&](int s0, auto f) {
        uint32_t sum = 0;
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
            if (s0 + k * kWave < p.S) sum += uint32_t(f(kv_span(p, len[k]).tiles));
        return sum;
    };
    auto sum_all = [&](auto f) {
        uint32_t sum = 0;
        for (int s0 = 0; s0 < p.S; s0 += kAll) {
            if (p.S > kAll) read(s0);
            sum += sum_read(s0, f);
        }
        return wave_sum(sum);
    };
    if (p.S <= kAll) read(0);
    const uint32_t total = sum_all([](int n) { return n; });
    auto size_of = [&](uint32_t shares) {
        const int size = int((total + shares - 1) / shares);
        return size > p.min_tiles ? size : p.min_tiles;
    };
    r.size = size_of(uint32_t(p.shares));
    bool apart = p.S == 1;                                   // no share holds tiles of two sequences
    if (!apart && p.S <= kAll) {
        auto shares_of = [&](int n) { return (n + r.size - 1) / r.size; };
        apart = sum_all(shares_of) <= uint32_t(p.shares);
        if (!apart) {
            const uint32_t some = sum_all([](int n) { return n > 0 ? 1 : 0; });
            if (8 * some <= uint32_t(p.shares)) {            // (at most a seventh more tiles a share)
                r.size = size_of(uint32_t(p.shares) - some);
                apart = true;
            }
        }
    }
    // in shares, or in tiles
    auto units_of = [&](int n) { return apart ? (n + r.size - 1) / r.size : n; };
    const int64_t wanted = apart ? int64_t(x) : int64_t(x) * r.size;
    if (!apart && wanted >= int64_t(total)) return false;
    int before = 0;
    for (int s0 = 0; s0 < p.S; s0 += kAll) {
        if (p.S > kAll) {
            read(s0);
            const int all = s0 + kAll < p.S ? int(wave_sum(sum_read(s0, units_of))) : 0;
            if (s0 + kAll < p.S && wanted >= int64_t(before) + all) {
                before += all;
                continue;
            }
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            if (s0 + k * kWave >= p.S) break;
            const int n = units_of(kv_span(p, len[k]).tiles), upto = sum_upto(n);
            const int all = __builtin_amdgcn_readlane(upto, kWave - 1);
            if (wanted < int64_t(before) + all) {
                const int at = __ffsll(static_cast<unsigned long long>(__ballot(before + upto > int(wanted)))) - 1;
                const int skipped = int(wanted) - (before + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
                r.seq = s0 + k * kWave + at;
                r.span = kv_span(p, __builtin_amdgcn_readlane(len[k], at));
                r.offset = apart ? skipped * r.size : skipped;
                const int rest = apart ? r.span.tiles - r.offset : int(total) - int(wanted);       // (the last share ends with the last tile)
                r.left = rest < r.size ? rest : r.size;
                return true;
            }
            before += all;
        }
    }
    return false;
}

template <int DT> __device__ __forceinline__ float4v kv_mfma(uint4v a, uint4v b, float4v c) {
    if constexpr (DT == FQ_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16v8, a), __builtin_bit_cast(bf16v8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ float low_value(uint32_t w) {
    if constexpr (DT == FQ_BF16) return bits_to_float(w << 16);
    else return f16_to_float(uint16_t(w & 0xffffu));
}
template <int DT> __device__ __forceinline__ float high_value(uint32_t w) {
    if constexpr (DT == FQ_BF16) return bits_to_float(w & 0xffff0000u);
    else return f16_to_float(uint16_t(w >> 16));
}

// HW heads of a workgroup, TW wavefronts of each; SHARED: a share of all tiles, else one sequence.
template <int D, int DT, int HW, int TW, bool SHARED>
__global__ __launch_bounds__(HW * TW * kWave) void paged_kv_decode_kernel(const KvDecodeParams p) {
    constexpr int KP = D / 64;                       // lines of 128 bytes of a key
    constexpr int VH = D == 256 ? 2 : 1;             // halves of 128 coordinates
    constexpr int VW = D == 64 ? 2 : 4;              // words of a lane's piece of a value row
    constexpr int VE = 2 * VW;                       // its coordinates
    constexpr int W = HW * TW;
    extern __shared__ __align__(16) float lds[];     // (W, G, D), then (W, 2, 16), then (HW, 16)
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n = lane & 15, g = lane >> 4, kgroup = (n >> 2) & 1;
    const int G = p.G;
    const int groups = p.H_KV / HW;                  // of HW neighbouring heads
    const int x = blockIdx.x / groups, head = (blockIdx.x - x * groups) * HW + wave % HW, turn = wave / HW;

    const uint16_t* kbase = p.kc + head * p.k_head + 8 * (g + 4 * (n >> 3)) + int64_t(n & 3) * p.k_token;
    const uint16_t* vbase = p.vc + head * p.v_head + VE * n;
    const int page_mask = (1 << p.page_log2) - 1;
    const int last_tile = ((p.max_blocks << p.page_log2) - 1) / kKvTile;

    // Where a wavefront's next 16 tiles lie: lane 4 i + b knows it of keys 8 b .. 8 b + 7 of the i-th (one load and one
    // multiplication a group of 8 keys; the tiles fetch it across lanes).  Bit 4 i + b of `present`: the page is one of the cache.
    int64_t key_at = 0, value_at = 0;
    uint64_t present = 0;
    auto token_of = [&](int tile) {                  // of lane 4 i + b, the i-th tile from `tile` on
        const int t = tile + TW * (lane >> 2);
        return (t < last_tile ? t : last_tile) * kKvTile + 8 * (lane & 3);
    };
    auto block_of = [&](const int32_t* table, int tile) {
        const int b = token_of(tile) >> p.page_log2;
        return table[b < p.max_blocks ? b : p.max_blocks - 1];
    };
    auto locate = [&](int tile, int block) {
        const bool in_cache = uint32_t(block) < uint32_t(p.num_blocks);
        present = __ballot(in_cache);
        const int b = in_cache ? block : 0, t = token_of(tile) & page_mask;
        key_at = int64_t(b) * p.k_block + int64_t(t) * p.k_token;
        value_at = int64_t(b) * p.v_block + int64_t(t) * p.v_token;
    };
    auto fetch = [&](int64_t v, int at) {            // from lane at / 4
        const int lo = __builtin_amdgcn_ds_bpermute(at, int(v)), hi = __builtin_amdgcn_ds_bpermute(at, int(v >> 32));
        return (int64_t(hi) << 32) | uint32_t(lo);
    };

    uint4v kr[2][2][KP];
    uint32_t vr[8][VH][VW];
    auto load_keys = [&](int i) {                    // of the i-th tile of the 16
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint16_t* src = kbase + fetch(key_at, 16 * i + 4 * kgroup + 8 * h);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int a = 0; a < KP; ++a) kr[t][h][a] = __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(src + 64 * a));
                src += 4 * p.k_token;
            }
        }
    };
    auto load_values = [&](int i) {
        const uint16_t* src = vbase + fetch(value_at, 16 * i + 4 * g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma unroll
            for (int h = 0; h < VH; ++h) {
                if constexpr (VW == 4) {
                    const uint4v w = __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(src + 128 * h));
                    vr[k][h][0] = w.x; vr[k][h][1] = w.y; vr[k][h][2] = w.z; vr[k][h][3] = w.w;
                } else {
                    const uint2v w = __builtin_nontemporal_load(reinterpret_cast<const uint2v*>(src));
                    vr[k][h][0] = w.x; vr[k][h][1] = w.y;
                }
            }
            src += p.v_token;
        }
    };

    int seq = x, offset = 0, left = 0;               // the sequence, its first tile here, the tiles left of the share
    KvPlace at;
    if constexpr (SHARED) {
        if (!(p.S <= kWave ? kv_place<1>(p, x, lane, at) : kv_place<8>(p, x, lane, at))) return;
        seq = at.seq;
        offset = at.offset;
        left = at.left;
    }
    bool again = false;
    do {
        const int32_t* table = p.table + int64_t(seq) * p.table_row;
        int block = 0;
        if (!SHARED && p.window == 0) block = block_of(table, turn);     // known before the length is
        uint4v qr[2 * KP];
        {
            const uint16_t* src = p.q + int64_t(seq) * p.q_seq + int64_t(head * G + (n < G ? n : 0)) * p.q_head + 8 * g;
#pragma unroll
            for (int j = 0; j < 2 * KP; ++j) qr[j] = *reinterpret_cast<const uint4v*>(src + 32 * j);
        }
        const KvSpan span = SHARED ? at.span : kv_span(p, p.lens[seq]);
        const int count = !SHARED || span.tiles - offset < left ? span.tiles - offset : left;
        const int end = span.first + offset + count;

        float4v acc[VH][VE];
#pragma unroll
        for (int h = 0; h < VH; ++h)
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[h][e] = float4v{0.f, 0.f, 0.f, 0.f};
        float m = -__builtin_inff(), l = 0.0f;

        int tile = span.first + offset + turn;
        if (tile < end) {
            if (SHARED || p.window != 0) block = block_of(table, tile);
            locate(tile, block);
            load_keys(0);
            load_values(0);
            int i = 0;                               // the tile's number among the 16
            int pages = int(present & 15);
            block = block_of(table, tile + 16 * TW);
#pragma unroll
            for (int j = 0; j < 2 * KP; ++j) qr[j] = n < G ? qr[j] : uint4v{0u, 0u, 0u, 0u};
            // (whether another tile follows is known at compile time: a branch round the loads would make the waits for
            // the values wait for the next keys as well)
            auto step = [&](auto followed) {
                constexpr bool more = decltype(followed)::value;
                float4v s[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float4v half[2][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            half[h][c] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int a = 0; a < KP; ++a) half[h][c] = kv_mfma<DT>(kr[t][h][a], qr[2 * a + c], half[h][c]);
                        }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t lo = float_to_bits(lane < 32 ? half[0][0][r] : half[0][1][r]);
                        const uint32_t hi = float_to_bits(lane < 32 ? half[1][0][r] : half[1][1][r]);
                        const auto both = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
                        s[t][r] = bits_to_float(both[0]) + bits_to_float(both[1]);
                    }
                }
                const int pages_now = pages;
                if constexpr (more) {
                    if (++i == 16) {
                        i = 0;
                        locate(tile + TW, block);
                        block = block_of(table, tile + 17 * TW);
                    }
                    pages = int(present >> (4 * i)) & 15;
                    load_keys(i);
                }
                __builtin_amdgcn_sched_barrier(0);
                float sv[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) sv[k] = s[k >> 2][k & 3] * p.scale_log2;
                // v_perm selectors that turn two keys' words into two coordinates' pairs of keys; a byte of 12 is a zero
                uint32_t even[4], odd[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) { even[k] = 0x05040100u; odd[k] = 0x07060302u; }
                // whole tiles whose pages are all in the cache need no mask
                if (pages_now != 15 || tile * kKvTile < span.lo || tile * kKvTile + kKvTile > span.len) {
                    const int key = tile * kKvTile + 8 * g;
                    int from = span.lo - key, to = span.len - key;
                    from = from < 0 ? 0 : from > 8 ? 8 : from;
                    to = to < 0 ? 0 : to > 8 ? 8 : to;
                    uint32_t seen = ((1u << to) - 1u) & ~((1u << from) - 1u);
                    seen = (pages_now >> g) & 1 ? seen : 0u;
#pragma unroll
                    for (int k = 0; k < 8; ++k) sv[k] = (seen >> k) & 1u ? sv[k] : -__builtin_inff();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t keep = ((seen >> (2 * k)) & 1u ? 0x0000ffffu : 0u) | ((seen >> (2 * k + 1)) & 1u ? 0xffff0000u : 0u);
                        even[k] = (even[k] & keep) | (0x0c0c0c0cu & ~keep);
                        odd[k] = (odd[k] & keep) | (0x0c0c0c0cu & ~keep);
                    }
                }
                float top = sv[0];
#pragma unroll
                for (int k = 1; k < 8; ++k) top = __builtin_fmaxf(top, sv[k]);
                top = max_xor32(max_xor16(top));
                if (__any(top > m)) {
                    const float higher = __builtin_fmaxf(m, top);
                    const float shrink = m == higher ? 1.0f : __builtin_amdgcn_exp2f(m - higher);
                    l *= shrink;
#pragma unroll
                    for (int h = 0; h < VH; ++h)
#pragma unroll
                        for (int e = 0; e < VE; ++e) acc[h][e] *= shrink;
                    m = higher;
                }
                const float ref = m == -__builtin_inff() ? 0.0f : m - kKvLift<DT>;
                uint4v hi, lo;
                float w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = __builtin_amdgcn_exp2f(sv[k] - ref);
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    hi[k / 2] = round_pair<DT>(w[k], w[k + 1]);
                    lo[k / 2] = round_pair<DT>(w[k] - low_value<DT>(hi[k / 2]), w[k + 1] - high_value<DT>(hi[k / 2]));
                }
                l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                // (all of this before the wait for the values)
                asm volatile("" : "+v"(hi), "+v"(lo), "+v"(l));
                uint4v vt[VH][VE];
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int e = 0; e < VE; ++e)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            vt[h][e][k] = __builtin_amdgcn_perm(vr[2 * k + 1][h][e / 2], vr[2 * k][h][e / 2], e & 1 ? odd[k] : even[k]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (more) load_values(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[h][e] = kv_mfma<DT>(vt[h][e], lo, acc[h][e]);
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[h][e] = kv_mfma<DT>(vt[h][e], hi, acc[h][e]);
            };
            for (; tile + TW < end; tile += TW) step(std::true_type{});
            step(std::false_type{});
            l = sum_xor32(sum_xor16(l));
        }

        const bool complete = !SHARED || count == span.tiles;
        if (SHARED && offset == 0 && threadIdx.x == 0 && int(blockIdx.x) == x * groups)
            p.place[seq] = int2{x, 1 + (span.tiles - count + at.size - 1) / at.size};
        const int64_t row = (int64_t(x + seq) * p.H_KV + head) * G;      // of the partial results
        const int64_t orow = (int64_t(seq) * p.H_KV + head) * G;         // of the outputs
        auto write_sum = [&](int h, float mt, float lt) {
            if (!complete) {
                p.part_m[row + h] = mt;
                p.part_l[row + h] = lt;
            } else if (p.lse != nullptr) {
                p.lse[orow + h] = lt == 0.0f ? -__builtin_inff() : (mt - kKvLift<DT> + __builtin_amdgcn_logf(lt)) * (1.0f / kLog2e);
            }
        };
        // lane (g, h) holds coordinates VE (4 g + r) + e of head h
        if constexpr (TW == 1) {
            if (n < G) {
                const float inv = inverse_sum(l);
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int c = 128 * h + VE * (4 * g + r);
#pragma unroll
                        for (int e = 0; e < VE; e += 4) {
                            if (complete)
                                *reinterpret_cast<uint2v*>(p.out + (orow + n) * D + c + e) =
                                    uint2v{round_pair<DT>(acc[h][e][r] * inv, acc[h][e + 1][r] * inv),
                                           round_pair<DT>(acc[h][e + 2][r] * inv, acc[h][e + 3][r] * inv)};
                            else
                                *reinterpret_cast<float4v*>(p.part_o + (row + n) * D + c + e) =
                                    float4v{acc[h][e][r], acc[h][e + 1][r], acc[h][e + 2][r], acc[h][e + 3][r]};
                        }
                    }
                if (g == 0) write_sum(n, m, l);
            }
        } else {
            // the wavefronts of a head are joined in LDS
            float* sm = lds + W * G * D;             // (W, 2, 16)
            if (SHARED && again) __syncthreads();    // the piece before has been read
            if (g == 0) {
                sm[wave * 32 + n] = m;
                sm[wave * 32 + 16 + n] = l;
            }
            __syncthreads();
            const int mine = wave % HW;
            float top = sm[mine * 32 + n];
#pragma unroll
            for (int w = 1; w < TW; ++w) top = __builtin_fmaxf(top, sm[(mine + w * HW) * 32 + n]);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < TW; ++w) {
                const float mw = sm[(mine + w * HW) * 32 + n], lw = sm[(mine + w * HW) * 32 + 16 + n];
                sum += lw * piece_weight(mw, lw, top);
            }
            float* scale = sm + W * 32;              // (HW, 16)
            if (turn == 0 && g == 0) {
                if (n < G) write_sum(n, top, sum);
                scale[mine * 16 + n] = complete ? inverse_sum(sum) : 1.0f;
            }
            const float weight = piece_weight(m, l, top);
            if (n < G) {
#pragma unroll
                for (int h = 0; h < VH; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float* dst = lds + (wave * G + n) * D + 128 * h + VE * (4 * g + r);
#pragma unroll
                        for (int e = 0; e < VE; e += 4)
                            *reinterpret_cast<float4v*>(dst + e) = float4v{acc[h][e][r] * weight, acc[h][e + 1][r] * weight,
                                                                           acc[h][e + 2][r] * weight, acc[h][e + 3][r] * weight};
                    }
            }
            __syncthreads();
            // the HW heads' rows lie side by side, in LDS and in memory
            for (int i = 4 * int(threadIdx.x); i < HW * G * D; i += 4 * W * kWave) {
                float4v o = *reinterpret_cast<const float4v*>(lds + i);
#pragma unroll
                for (int w = 1; w < TW; ++w) o += *reinterpret_cast<const float4v*>(lds + w * HW * G * D + i);
                const int h = i / D;
                const float inv = scale[h / G * 16 + h % G];
                const int64_t at = i - int64_t(mine) * G * D;        // from this wavefront's head on
                if (complete)
                    *reinterpret_cast<uint2v*>(p.out + orow * D + at) = uint2v{round_pair<DT>(o.x * inv, o.y * inv), round_pair<DT>(o.z * inv, o.w * inv)};
                else
                    *reinterpret_cast<float4v*>(p.part_o + row * D + at) = o;
            }
        }
        if constexpr (SHARED) {
            left -= count;
            offset = 0;
            again = true;
            // the next sequence that has tokens (the rows of those without: the second launch)
            if (left > 0) {
                uint64_t some = 0;
                for (++seq; some == 0 && seq < p.S; seq += some == 0 ? kWave : 0) {
                    const int len = kv_len_of(p, seq + lane);
                    some = __ballot(kv_span(p, len).tiles > 0);
                    if (some != 0) {
                        const int first = __ffsll(static_cast<unsigned long long>(some)) - 1;
                        at.span = kv_span(p, __builtin_amdgcn_readlane(len, first));
                        seq += first;
                    }
                }
            }
        }
    } while (SHARED && left > 0 && seq < p.S);
}

// Joins the pieces of the sequences that several shares hold, and writes the rows of those that have no tokens.  A workgroup
// takes 4 Q neighbouring values of the G rows of one sequence and KV head, R pieces at a time, each thread with a maximum and a
// sum of its own (so one trip to memory brings all it needs).
template <int D, int DT, int Q>
__global__ __launch_bounds__(256) void paged_kv_join_kernel(const KvDecodeParams p) {
    constexpr int R = 256 / Q;
    __shared__ __align__(16) float4v rows[R][Q];
    __shared__ float2v sums[R][Q];
    const int columns = p.G * D / (4 * Q);
    const int64_t group = blockIdx.x / columns;                          // sequence and KV head
    const int seq = int(group / p.H_KV);
    const int c = 4 * (int(blockIdx.x % columns) * Q + threadIdx.x % Q), r0 = threadIdx.x / Q, h = c / D;
    const int2 place = p.place[seq];
    const int share0 = place.x, pieces = kv_span(p, p.lens[seq]).tiles > 0 ? place.y : 0;   // (of sequences without tokens nothing is written)
    if (pieces == 1) return;
    const int64_t step = int64_t(p.H_KV) * p.G;                          // rows from one piece to the next
    const int64_t first = int64_t(share0 + seq) * step + (group - int64_t(seq) * p.H_KV) * p.G;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.0f;
    auto take = [&](float4v v, float m, float l) {
        const float higher = __builtin_fmaxf(top, m);
        const float a = piece_weight(top, sum, higher), b = piece_weight(m, l, higher);
        o = o * a + v * b;
        sum = sum * a + l * b;
        top = higher;
    };
    if (pieces <= R) {                                                   // (most sequences: one trip, nothing read twice)
        if (r0 < pieces) {
            const int64_t row = first + r0 * step;
            o = *reinterpret_cast<const float4v*>(p.part_o + row * D + c);
            top = p.part_m[row + h];
            sum = p.part_l[row + h];
        }
    } else {
        for (int i = r0; i < pieces; i += 4 * R) {                       // four pieces a trip
            float4v v[4];
            float m[4], l[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t row = first + (i + k * R < pieces ? i + k * R : i) * step;
                v[k] = *reinterpret_cast<const float4v*>(p.part_o + row * D + c);
                m[k] = p.part_m[row + h];
                l[k] = p.part_l[row + h];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * R < pieces) take(v[k], m[k], l[k]);
        }
    }
    // the R rows' results, weighed against the highest maximum and added (a row without pieces has a sum of zero, so weight 0)
    const int q = threadIdx.x % Q;
    sums[r0][q] = float2v{top, sum};
    __syncthreads();
    float highest = -__builtin_inff(), den = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) highest = __builtin_fmaxf(highest, sums[r][q].x);
#pragma unroll
    for (int r = 0; r < R; ++r) den += sums[r][q].y * piece_weight(sums[r][q].x, sums[r][q].y, highest);
    rows[r0][q] = o * piece_weight(top, sum, highest);
    __syncthreads();
    if (threadIdx.x < Q) {
        float4v all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < R; ++r) all += rows[r][q];
        const float inv = inverse_sum(den);
        const int64_t out = group * p.G;
        *reinterpret_cast<uint2v*>(p.out + out * D + c) = uint2v{round_pair<DT>(all.x * inv, all.y * inv), round_pair<DT>(all.z * inv, all.w * inv)};
        if (c % D == 0 && p.lse != nullptr)
            p.lse[out + h] = den == 0.0f ? -__builtin_inff() : (highest - kKvLift<DT> + __builtin_amdgcn_logf(den)) * (1.0f / kLog2e);
    }
}

}  // namespace fq

namespace {

// How a call is divided.
struct KvPlan {
    int shares;          // workgroups among which the tiles of a KV head are divided; 0: one a sequence, and no second launch
    int heads, waves;    // KV heads of a workgroup, wavefronts of each
};

// The host knows the table's width, not the lengths, and divides for sequences that fill it.  All times below are of tables as wide as
// the longest sequence; in wider ones short sequences are divided where that costs (tables for 4096 and for 131072 tokens: 1 x 777 8.9 and
// 10.1 us, 10 x 430 12.2 and 12.2, 16 x 500 13.8 and 13.8, 32 x 1000 26.9 and 27.1).
// Undivided sequences or shares: a CU takes its tiles at 40 to 60 GB/s, so few long sequences have to be spread, but the second
// launch costs 3 us, and a share that goes on with another sequence starts from nothing again (3 us; asking for that one's
// pages ahead was no faster).  In us, undivided / shares, 32 heads over 8, bf16:
//   of 128: 1 x 200 tokens 6.1 / 9.1, 1 x 430 9.1 / 9.3, 1 x 777 11.1 / 9.2, 1 x 2000 28.3 / 10.4, 10 x 430 10.0 / 12.6, 10 x 700 13.5 / 13.3,
//     16 x 500 12.2 / 14.1, 16 x 1000 18.5 / 18.4, 32 x 1000 25.0 / 27.2, 32 x 2000 45.7 / 47.9, 64 x 1000 47.4 / 48.5, 200 of 100 to 2000
//     181 / 159; 8 heads over 1: 10 x 700 12.1 / 10.1, 32 of 100 to 700 11.7 / 10.4, 128 of them 13.0 / 14.1, 64 of 200 to 1500 20.1 / 13.5,
//     300 of them 30.7 / 34.3; 16 over 2, 60 of 200 to 700 13.2 / 15.6; 32 over 32, 16 of 300 to 1000 38.9 / 36.6
//   of 64: 1 x 640 7.1 / 8.4, 10 x 700 9.9 / 11.3, 64 x 500 15.7 / 17.7, 64 of 300 to 1000 20.7 / 20.1
//   of 256: 1 x 200 9.4 / 11.5, 1 x 300 11.6 / 11.6, 1 x 430 14.5 / 11.6, 10 x 300 12.2 / 14.2, 10 x 700 21.2 / 18.5, 30 x 700 30.7 / 36.1.
// Eight wavefronts of one head have few tiles of a sequence each, so there a share that goes on costs most: 8 heads over 1, 600 of 100 to
// 1200 43 / 49 (of 64: 24 / 33; of 256: 80 / 82), 1500 of 100 to 2000 138 / 150, 600 of 100 to 3500 103 / 99 (of 256: 204 /
// 188); 16 over 2, 1000 of 100 to 1200 127 / 125.
// The workgroup: four heads and two wavefronts of each draw best where there is much (see above); where a call has at most two
// tiles for every wavefront of the card, two heads of two, of which a CU has two, spread it further: 1 x 1000 12.2 -> 10.1 us,
// 1 x 4000 13.6 -> 12.0, 8 heads over 1, 4 x 1500 14.6 -> 12.6; but 61 of 500 to 16000 343 -> 355.
// tables of so many tiles are never divided
int kv_whole_tiles(int D) { return D == 256 ? 10 : D == 128 ? 14 : 24; }
KvPlan kv_plan(int S, int H_KV, int D, int64_t max_tokens, int window) {
    int64_t tiles = (max_tokens + fq::kKvTile - 1) / fq::kKvTile;
    if (window > 0 && window / fq::kKvTile + 2 < tiles) tiles = window / fq::kKvTile + 2;
    const int64_t whole = int64_t(S) * H_KV, cus = fq_host::device_cu_count();
    const int together = H_KV % 4 == 0 ? 4 : H_KV % 2 == 0 ? 2 : 1, most = D == 256 ? 4 : 8;
    KvPlan r = {0, 1, most};
    const int middle = D == 256 ? 12 : 25;
    if (tiles <= kv_whole_tiles(D) || (tiles <= middle && 8 * whole >= 3 * cus) || (tiles <= 64 && whole >= cus / 2 && whole < 2 * cus) ||
        (together == 1 && D != 256 && tiles <= 80 && whole >= 2 * cus) || int64_t(S) * tiles >= (1LL << 31)) {                 // (more tiles than are counted)
        if (together == 4 && whole >= 8 * cus) {
            // fewer workgroups: 256 of 50 to 300 tokens, 32 heads over 8 of 128, 40 us; 52 with a head a workgroup
            r.heads = 4;
            r.waves = most / 4;
        }
        return r;
    }
    const bool few = D != 256 && whole * tiles <= 16 * cus;
    r.heads = few && together == 4 ? 2 : together;
    r.waves = (few ? 4 : most) / r.heads;
    // as many workgroups as run at a time: more are no faster (two rounds, 32 x 4096: 86.7 -> 96 us)
    r.shares = int(((few ? 2 : 1) * cus * r.heads + H_KV - 1) / H_KV);
    return r;
}
// the most shares of any of these plans, and of those for a window
int kv_most_shares(int H_KV) { return int((4 * int64_t(fq_host::device_cu_count()) + H_KV - 1) / H_KV); }

int check_kv_shape(int S, int H_Q, int H_KV, int D, int block_size, int max_blocks, int64_t num_blocks) {
    if (S < 0 || H_Q <= 0 || H_KV <= 0 || max_blocks <= 0 || num_blocks <= 0) return FQ_ERR_BAD_SHAPE;
    if (!fq_host::supported_dim(D)) return FQ_ERR_UNSUPPORTED_DIM;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (H_Q % H_KV != 0 || H_Q / H_KV > 16) return FQ_ERR_BAD_SHAPE;
    if (num_blocks > 0x7fffffffLL || int64_t(max_blocks) * block_size > 0x7fffffe0LL) return FQ_ERR_BAD_SHAPE;
    return FQ_OK;
}

size_t round_up(size_t n) { return (n + 255) & ~size_t(255); }

struct KvRoom {
    size_t o, m, place, all;
};
KvRoom kv_room(int S, int H_Q, int D, int shares) {
    const size_t rows = (size_t(S) + size_t(shares)) * size_t(H_Q);
    KvRoom r;
    r.o = round_up(rows * size_t(D) * 4);
    r.m = round_up(rows * 4);
    r.place = round_up(size_t(S) * sizeof(int2));
    r.all = shares == 0 ? 0 : r.o + 2 * r.m + r.place;
    return r;
}

template <int D, int DT, int HW, int TW, bool SHARED>
int launch_attend(const fq::KvDecodeParams& p, hipStream_t s) {
    const size_t lds = TW == 1 ? 0 : (size_t(HW * TW) * p.G * D + HW * TW * 32 + HW * 16) * 4;
    auto kernel = fq::paged_kv_decode_kernel<D, DT, HW, TW, SHARED>;
    if (lds > 32768 && !fq_host::lds_limit_raised(reinterpret_cast<const void*>(kernel), lds)) return FQ_ERR_LAUNCH;
    kernel<<<unsigned(SHARED ? p.shares : p.S) * unsigned(p.H_KV / HW), HW * TW * 64, lds, s>>>(p);
    return FQ_OK;
}

template <int D, int DT>
int launch_kv(const fq::KvDecodeParams& p, const KvPlan& plan, hipStream_t s) {
    constexpr int W = D == 256 ? 4 : 8;
    int st;
    if (plan.shares > 0) {
        if (plan.heads == 4) st = launch_attend<D, DT, 4, W / 4, true>(p, s);
        else if (plan.heads == 2) st = plan.waves == W / 2 ? launch_attend<D, DT, 2, W / 2, true>(p, s) : launch_attend<D, DT, 2, 2, true>(p, s);
        else st = plan.waves == W ? launch_attend<D, DT, 1, W, true>(p, s) : launch_attend<D, DT, 1, 4, true>(p, s);
        if (st != FQ_OK) return st;
        // as many values a workgroup as leave enough workgroups
        const int64_t values = int64_t(p.S) * p.H_KV * p.G * D;
        if (p.G * D % 256 == 0 && values / 256 >= 2 * fq_host::device_cu_count())
            fq::paged_kv_join_kernel<D, DT, 64><<<unsigned(values / 256), 256, 0, s>>>(p);
        else
            fq::paged_kv_join_kernel<D, DT, 16><<<unsigned(values / 64), 256, 0, s>>>(p);
    } else if (plan.heads == 4) {
        st = launch_attend<D, DT, 4, W / 4, false>(p, s);
    } else {
        st = launch_attend<D, DT, 1, W, false>(p, s);
    }
    return st != FQ_OK ? st : fq_host::check_launch();
}

template <int D>
int launch_kv_type(const fq::KvDecodeParams& p, const KvPlan& plan, int dtype, hipStream_t s) {
    return dtype == FQ_BF16 ? launch_kv<D, FQ_BF16>(p, plan, s) : launch_kv<D, FQ_F16>(p, plan, s);
}

}  // namespace

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
    const KvPlan plan = kv_plan(num_seqs, H_KV, D, int64_t(max_blocks_per_seq) * block_size, window);
    const int most = plan.shares == 0 ? 0 : kv_most_shares(H_KV);
    if ((int64_t(num_seqs) + most) * H_Q * (D / 32) > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    const KvRoom room = kv_room(num_seqs, H_Q, D, most);
    if (room.all > 0) {
        if (!workspace || workspace_bytes < room.all) return FQ_ERR_WORKSPACE;
        if (!fq_host::aligned(workspace, 256)) return FQ_ERR_MISALIGNED;
    }
    fq::KvDecodeParams p;
    p.q = static_cast<const uint16_t*>(q);
    p.kc = static_cast<const uint16_t*>(key_cache);
    p.vc = static_cast<const uint16_t*>(value_cache);
    p.table = block_table;
    p.lens = seq_lens;
    p.out = static_cast<uint16_t*>(out);
    p.lse = lse;
    char* ws = static_cast<char*>(workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_m = reinterpret_cast<float*>(ws + room.o);
    p.part_l = reinterpret_cast<float*>(ws + room.o + room.m);
    p.place = reinterpret_cast<int2*>(ws + room.o + 2 * room.m);
    p.q_seq = q_strides[0]; p.q_head = q_strides[1];
    p.k_block = key_strides[0]; p.k_token = key_strides[1]; p.k_head = key_strides[2];
    p.v_block = value_strides[0]; p.v_token = value_strides[1]; p.v_head = value_strides[2];
    p.table_row = block_table_stride;
    p.S = num_seqs; p.H_KV = H_KV; p.G = H_Q / H_KV;
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.max_blocks = max_blocks_per_seq; p.num_blocks = int(num_blocks); p.window = window;
    p.shares = plan.shares; p.min_tiles = plan.waves;        // a tile a wavefront
    p.scale_log2 = sm_scale * fq::kLog2e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_kv_type<64>(p, plan, dtype, s);
        case 128: return launch_kv_type<128>(p, plan, dtype, s);
        default: return launch_kv_type<256>(p, plan, dtype, s);
    }
}
