// Attention of one new token per sequence where sequences begin with the same pages: the keys of a shared prefix are read once for all
// queries that see them, what every sequence has behind it is read as in fq_paged_kv_decode.hpp, and the parts are joined by their
// maxima and sums:
//
//   o = (sum_{j in prefix} p_j v_j + sum_{j behind} p_j v_j) / (sum_{j in prefix} p_j + sum_{j behind} p_j)
//
// Members of prefix i are the sequences whose id it is and that are as long as it; no lists of them are asked for, and nothing on the
// host knows a length: every workgroup counts members and tiles for itself, with all lengths and ids asked for at once.
//
// What bounds it: the own tokens HBM, the prefix each wavefront's chain of scores, maximum, weights and products.  One launch has
// workgroups of both, and a second one joins.  At D 64 and 128 a CU has one of each, so that the ones' waits for memory and the others'
// products overlap (96 sequences behind 6000 tokens, 128, whole calls: the prefix alone 33 us, 50 to 1200 tokens each of their own 48,
// both 63).  At 256 a wavefront has 447 to 457 registers and a CU one workgroup: the prefixes', which come first, and then the others
// (47, 50, both 92).
//   * 128 rows (member, query head of the KV head), 32 a wavefront, against tiles of 16 KB of keys and as many of values in LDS,
//     double buffered, one barrier a tile.  S^T = K Q^T and O^T = V^T P on v_mfma_f32_32x32x16, rows along the columns: a lane's
//     scores are its own P operand, maximum and sum of a row two lanes' own.
//   * Every thread brings eight coordinates of eight tokens through registers, asked for a tile ahead: half of the threads keys, as they are,
//     16-byte pieces swizzled so that lanes reading one piece of 16 keys reach all banks; half of them values, turned (half a v_perm_b32 an
//     element) into operands.  Codes become 16-bit on the way.
//   * A tile takes 1.6 us on one workgroup a CU, fp16 over codes 1.8 (256 sequences behind 8192 and 16384 tokens; matrix cores busy 29 % of
//     the cycles, LDS 16, vector units 34).  Two of the prefixes' on a CU were no gain (with one term of a weight, see below, 4.3 us for two
//     tiles where one took 1.8, and a second prologue).  Scores of the next tile under the weights of this one need more registers than
//     two workgroups leave (300 spilled; as it is, at 128, 4 or 5 of 256).  Weights of 16 tokens run under the products of the 16 before
//     them, whose values are read before that (with this 31.2 -> 28.0 us at 40 sequences behind 32768 tokens).
//   * Weights go to the second product as two 16-bit terms (16 significant bits and more), as over a sequence's own tokens; the sums are of
//     the unrounded ones.  With one term a bf16 result was off by up to another 2^-8 of what was summed (0.0020 in the mean against 64
//     bits, where its own rounding is 0.0017); the second costs 256 sequences behind 8192 tokens 69 -> 76 us, 96 behind 6000 61 -> 62.
// Measured (whole calls): 96 sequences of 50 to 1200 tokens behind 6000, 32 heads over 8 of 128, bf16, 63 us (every sequence by
// itself 298); 150 of up to 900 behind three prefixes of 2848 to 5728 or none, 64 over 8, fp16 over 8 bits, 72 us (219); 40 behind 32768,
// 8 over 1, 8 bits, 29 us (59); 6 behind 2000 15 us (16); 64 of up to 600 behind two of 3000 to 4000, 32 over 8 of 64, 22 us (69), 8 bits
// 21 (41); 40 of them behind two of 2000 to 3000, 16 over 4 of 256, 36 us (71), 8 bits 34 (42).  It does not pay where sequences have
// much more of their own than they share: 50 of 8000 behind 2000 287 us (285), 8 bits 167 (155); nor for one or two a prefix, as a tile
// takes as long for four rows as for 128.
#include "fq_paged_kv_decode.hpp"

namespace fq {

struct PrefixParams {
    KvDecodeParams kv;
    int4* place;                          // (S): first piece of a member's prefix, pieces, row in each, unused
    int64_t first_row;                    // of the prefixes' partial results, behind those of the sequences' own tokens
    int shares, min_tiles;                // among which a KV head's work is divided
    int members;                          // of a workgroup's rows
};

constexpr int kPrefixRows = 128;
constexpr int kPrefixMost = 1024;         // prefixes of a call
constexpr int kPrefixSeqs = 1024;         // sequences whose prefixes are kept in LDS (the others' are read again)

template <int D> struct PrefixCfg {
    static constexpr int TT = 8192 / D;                    // tokens of a tile
    static constexpr int NB = TT / 32, NKS = D / 16, NOB = D / 32, NU = TT / 16, NG = TT / 8;
    static constexpr int SIDE = TT * D * 2;                // bytes of a tile's keys or values: 16 KB
    static constexpr int LDS = 4 * SIDE + 2 * TT * 4 + kPrefixRows * 4 + 3 * kPrefixMost * 4 + kPrefixSeqs * 2;
};

// Where a key's 16-byte pieces lie in its row of LDS, so that lanes that read one piece of 16 neighbouring keys reach all banks.
template <int D> __device__ __forceinline__ int key_swizzle(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }

template <int DT> __device__ __forceinline__ float16v wide_mfma(uint4v a, uint4v b, float16v c) {
    if constexpr (DT == FQ_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16v8, a), __builtin_bit_cast(bf16v8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// The members of a prefix, 128 rows (member, query head of the KV head) of them a workgroup, against a share of its keys.
template <int D, int DT, bool F8>
__device__ __forceinline__ void prefix_workgroup(const PrefixParams& pp, int workgroup, uint8_t* lds) {
    using C = PrefixCfg<D>;
    using Elem = std::conditional_t<F8, uint8_t, uint16_t>;
    constexpr int TT = C::TT, NB = C::NB, NKS = C::NKS, NOB = C::NOB, NU = C::NU, NG = C::NG;
    constexpr int PT = F8 ? FQ_BF16 : DT;                  // of weights and values in the second product
    constexpr bool POWERS = F8 && DT == FQ_F16;            // fp16 has no room for the powers of the rows: see keep()
    const KvDecodeParams& p = pp.kv;
    uint8_t *lk = lds, *lv = lds + 2 * C::SIDE;
    float* powers = reinterpret_cast<float*>(lds + 4 * C::SIDE);          // (2, 2, TT / 2), see keep()
    int* list = reinterpret_cast<int*>(powers + 2 * TT);                  // the sequences of the rows
    const int tid = threadIdx.x, lane = tid & 63, m32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = workgroup % p.H_KV, x = workgroup / p.H_KV, G = p.G;

    // ---- the share: members of every prefix, tiles of all, where this one begins -----------------------------------------------
    // (all lengths and ids are asked for at once; what the sequences share is kept in LDS for the lists of members)
    int* count = list + kPrefixRows;
    int* shared_len = count + kPrefixMost;
    int* leader = shared_len + kPrefixMost;                // the first of its members
    int16_t* shares_of = reinterpret_cast<int16_t*>(leader + kPrefixMost);
    constexpr int kAhead = 4;
    int ids[kAhead], lens[kAhead];
    auto ask = [&](int s0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int s = s0 + 256 * j + tid;
            ids[j] = -1;
            lens[j] = 0;
            if (s < p.S) {
                ids[j] = p.prefix_ids[s];
                lens[j] = p.lens[s];
            }
        }
    };
    ask(0);
    for (int i = tid; i < p.num_prefixes; i += 256) {
        count[i] = 0;
        leader[i] = p.S;
        const int n = p.prefix_lens[i] >> p.page_log2 << p.page_log2;
        shared_len[i] = n > 0 ? n : 0;
    }
    __syncthreads();
    const int64_t room = int64_t(p.max_blocks) << p.page_log2;
    auto prefix_of = [&](int id, int len) {                // that a sequence shares, or -1
        if (uint32_t(id) >= uint32_t(p.num_prefixes)) return -1;
        const int n = shared_len[id];
        return n > 0 && n <= (len > room ? room : int64_t(len)) ? id : -1;
    };
    for (int s0 = 0; s0 < p.S; s0 += 256 * kAhead) {
        if (s0 > 0) ask(s0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int s = s0 + 256 * j + tid, id = prefix_of(ids[j], lens[j]);
            if (s < kPrefixSeqs && s < p.S) shares_of[s] = int16_t(id);
            if (id >= 0) {
                atomicAdd(&count[id], 1);
                atomicMin(&leader[id], s);
            }
        }
    }
    __syncthreads();
    auto tiles_of = [&](int i) { return (shared_len[i] + TT - 1) / TT; };
    auto groups_of = [&](int i) { return int(uint32_t(count[i] + pp.members - 1) / uint32_t(pp.members)); };
    // in tiles, or in shares of `each` tiles that end with their group of rows (the host bounds the sum of either)
    auto units_of = [&](int i, int each) { return i < p.num_prefixes ? (tiles_of(i) + each - 1) / each * groups_of(i) : 0; };
    auto sum_of = [&](int each) {
        uint32_t sum = 0;
        for (int i0 = 0; i0 < p.num_prefixes; i0 += kWave) sum += wave_sum(uint32_t(units_of(i0 + lane, each)));
        return sum;
    };
    const uint32_t total = sum_of(1);
    int size = int((total + uint32_t(pp.shares) - 1) / uint32_t(pp.shares)), each = 1;
    if (size < pp.min_tiles) size = pp.min_tiles;
    // A share that goes on into another group takes as long as with four tiles more: better is one of up to three more, if all then end with
    // their groups (150 sequences behind three prefixes, 8 bits, 72 -> 68 us; 128 of 50 tokens behind 4096, whose shares end so anyway,
    // 31.2 -> 31.7: the sums).
    uint32_t pieces = 0;
    for (int n = size; each == 1 && n < size + 4; ++n) {
        pieces = sum_of(n);
        if (pieces <= uint32_t(pp.shares)) each = n;
    }
    if (each > 1) size = each;
    const int64_t begin = each > 1 ? x : int64_t(x) * size;
    if (begin >= int64_t(each > 1 ? pieces : total)) return;
    const int wanted = int(begin);
    int left = each > 1 || int(total) - wanted > size ? size : int(total) - wanted;
    int prefix = 0, group = 0, tile0 = 0, piece = x;       // piece: the share and the groups of rows before this one
    for (int i0 = 0, before = 0; i0 < p.num_prefixes; i0 += kWave) {
        const int units = units_of(i0 + lane, each), gs = units > 0 ? groups_of(i0 + lane) : 0;
        const int upto = before + sum_upto(units), groups_upto = sum_upto(gs);
        const uint64_t past = __ballot(upto > wanted);
        if (past != 0) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            prefix = i0 + at;
            const int inside = wanted - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(units, at));
            const int tiles = __builtin_amdgcn_readfirstlane(tiles_of(prefix)), per = (tiles + each - 1) / each;
            group = inside / per;
            tile0 = (inside - group * per) * each;
            if (each > 1 && left > tiles - tile0) left = tiles - tile0;
            piece += __builtin_amdgcn_readlane(groups_upto, at) - __builtin_amdgcn_readlane(gs, at) + group;
            break;
        }
        piece += __builtin_amdgcn_readlane(groups_upto, kWave - 1);
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }

    // ---- what this thread brings of a tile: eight coordinates of eight tokens; the first two wavefronts values, in the order of the
    // scores' registers, the others keys -----------------------------------------------------------------------------------------
    const bool brings_values = w < 2;
    const int item = tid & 127, igroup = item / (D / 8), ic = item % (D / 8);
    const int token0 = brings_values ? 16 * (igroup >> 1) + 4 * (igroup & 1) : 8 * igroup, token1 = token0 + (brings_values ? 8 : 4);    // four from each
    const int page_mask = (1 << p.page_log2) - 1;
    const Elem* base = static_cast<const Elem*>(brings_values ? p.vc : p.kc) + head * (brings_values ? p.v_head : p.k_head) + 8 * ic;
    const int64_t block_step = brings_values ? p.v_block : p.k_block, token_step = brings_values ? p.v_token : p.k_token;
    const uint8_t* scale_base = F8 ? (brings_values ? p.vs + head * p.vs_head : p.ks + head * p.ks_head) : nullptr;
    const int64_t scale_block = brings_values ? p.vs_block : p.ks_block;

    for (;;) {
        const int n_members = __builtin_amdgcn_readfirstlane(count[prefix]), shared = __builtin_amdgcn_readfirstlane(shared_len[prefix]);
        const int tiles = (shared + TT - 1) / TT, groups = int(uint32_t(n_members + pp.members - 1) / uint32_t(pp.members));
        const int here = left < tiles - tile0 ? left : tiles - tile0, end = tile0 + here;
        const int32_t* table = p.table + int64_t(__builtin_amdgcn_readfirstlane(leader[prefix])) * p.table_row;
        const int blocks = shared >> p.page_log2;
        // The pages of kAhead tiles, lane NG j + i that of the j-th tile's i-th eight tokens (-1: none of the cache), and those of the next ones.
        constexpr int kAhead = kWave / NG;
        auto entry_of = [&](int tile) { return ((tile + lane / NG) * TT + 8 * (lane % NG)) >> p.page_log2; };
        auto read_entries = [&](int tile) {
            const int b = entry_of(tile);
            return table[b < blocks ? b : blocks - 1];
        };
        auto pages_of = [&](int tile, int block) {
            return tile + lane / NG < end && entry_of(tile) < blocks && uint32_t(block) < uint32_t(p.num_blocks) ? block : -1;
        };
        const int first_entries = read_entries(tile0);
        // the group's members, in the order of the sequences
        if (w == 0) {
            int rank = 0;
            const int first = group * pp.members;
            for (int s0 = 0; s0 < p.S && rank < first + pp.members; s0 += kWave) {
                const int s = s0 + lane;
                const bool mine = s < p.S && (s < kPrefixSeqs ? int(shares_of[s]) : prefix_of(p.prefix_ids[s], p.lens[s])) == prefix;
                const uint64_t all = __ballot(mine);
                const int at = rank + __popcll(all & ((uint64_t(1) << lane) - 1)) - first;
                if (mine && at >= 0 && at < pp.members) list[at] = s;
                rank += __popcll(all);
            }
        }
        __syncthreads();
        const int members = n_members - group * pp.members < pp.members ? n_members - group * pp.members : pp.members;
        const int rows = members * G;
        if (tile0 == 0 && head == 0 && tid < members) pp.place[list[tid]] = int4{piece, 1 + (tiles - here + size - 1) / size, tid * G, 0};
        const int row = 32 * w + m32;
        const bool live = 32 * w < rows;
        uint4v qb[NKS];
        {
            const int r = row < rows ? row : 0;
            const uint16_t* src = p.q + int64_t(list[r / G]) * p.q_seq + int64_t(head * G + r % G) * p.q_head + 8 * hf;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) qb[ks] = *reinterpret_cast<const uint4v*>(src + 16 * ks);
            // scores are compared before they are scaled: a negative scale goes to the query, one of zero makes it zero
            if (!POWERS && !(p.scale_log2 > 0.0f)) {
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) qb[ks] = p.scale_log2 == 0.0f ? uint4v{0u, 0u, 0u, 0u} : qb[ks] ^ 0x80008000u;
            }
        }
        const float scale = p.scale_log2 == 0.0f ? 1.0f : (F8 ? 2.0f : 1.0f) * __builtin_fabsf(p.scale_log2);       // (codes: half keys)

        int pages = pages_of(tile0, first_entries), next = read_entries(tile0 + kAhead), asked = 0;      // asked: the number in `pages` of the tile asked for next
        constexpr int NW = F8 ? 2 : 4;                     // words of eight coordinates
        struct Part {
            uint32_t word[8][NW];
            uint32_t scales[2];
            uint32_t there;                                // which eights of the tile are in the cache
        };
        Part part;
        auto load = [&](int tile) __attribute__((always_inline)) {      // (no branch round the loads, so that nothing waits for them here)
            part.there = uint32_t(__ballot(pages >= 0) >> (NG * asked)) & ((1u << NG) - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int token = h ? token1 : token0, block = __builtin_amdgcn_ds_bpermute(4 * (NG * asked + token / 8), pages);
                const int b = block < 0 ? 0 : block, t = (tile * TT + token) & page_mask;
                const Elem* src = base + int64_t(b) * block_step + int64_t(t) * token_step;
#pragma unroll
                for (int i = 4 * h; i < 4 * h + 4; ++i) {
                    if constexpr (F8) {
                        const uint2v v = *reinterpret_cast<const uint2v*>(src);
                        part.word[i][0] = v.x; part.word[i][1] = v.y;
                    } else {
                        const uint4v v = *reinterpret_cast<const uint4v*>(src);
                        part.word[i][0] = v.x; part.word[i][1] = v.y; part.word[i][2] = v.z; part.word[i][3] = v.w;
                    }
                    src += token_step;
                }
                if constexpr (F8) part.scales[h] = *reinterpret_cast<const uint32_t*>(scale_base + int64_t(b) * scale_block + t);
            }
            if (++asked == kAhead) {
                asked = 0;
                pages = pages_of(tile + 1, next);
                next = read_entries(tile + 1 + kAhead);
            }
        };
        // Into LDS, as the products read them.  Codes become bfloat16 with half the powers of their rows, exactly (half: a code may stand for
        // 2^128); keys that meet fp16 queries become fp16 without them, as exactly, and the powers are applied to the scores in float32.
        auto keep = [&](int buffer) __attribute__((always_inline)) {
            uint32_t word[8][4];
            if constexpr (F8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t bits = part.scales[h];
                    const float up[4] = {row_scale<0>(bits), row_scale<1>(bits), row_scale<2>(bits), row_scale<3>(bits)};
                    if (POWERS && !brings_values) {
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                word[4 * h + t][2 * i] = codes_pair<DT, false>(part.word[4 * h + t][i]);
                                word[4 * h + t][2 * i + 1] = codes_pair<DT, true>(part.word[4 * h + t][i]);
                            }
                        // tokens 8 i + 4 hf + 0 .. 3 at place (hf, i)
                        if (ic == 0) {
                            const int four = (h ? token1 : token0) / 4;
                            *reinterpret_cast<float4v*>(powers + buffer * TT + 4 * ((four & 1) * NG + (four >> 1))) =
                                float4v{p.scale_log2 * up[0], p.scale_log2 * up[1], p.scale_log2 * up[2], p.scale_log2 * up[3]};
                        }
                    } else {
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t codes = part.word[4 * h + t][i];
                                word[4 * h + t][2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 0.5f * up[t], false));
                                word[4 * h + t][2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 0.5f * up[t], true));
                            }
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) word[t][i] = part.word[t][i % NW];
            }
            if (brings_values) {
                if (part.there != (1u << NG) - 1) {        // (a weight of 0 times what lies there must be 0)
#pragma unroll
                    for (int t = 0; t < 8; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) word[t][i] = (part.there >> ((t < 4 ? token0 : token1) / 8)) & 1 ? word[t][i] : 0u;
                }
                uint8_t* dst = lv + buffer * C::SIDE + ((igroup >> 1) * NOB + (ic >> 2)) * 1024 + (igroup & 1) * 512 + (ic & 3) * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint4v o;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[i] = __builtin_amdgcn_perm(word[2 * i + 1][c / 2], word[2 * i][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
                    *reinterpret_cast<uint4v*>(dst + 16 * (c ^ (ic & 7))) = o;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = token0 + i;
                    *reinterpret_cast<uint4v*>(lk + buffer * C::SIDE + r * (2 * D) + 16 * (ic ^ key_swizzle<D>(r))) = uint4v{word[i][0], word[i][1], word[i][2], word[i][3]};
                }
            }
        };

        float16v O[NOB];
#pragma unroll
        for (int ob = 0; ob < NOB; ++ob)
#pragma unroll
            for (int e = 0; e < 16; ++e) O[ob][e] = 0.0f;
        float m = -__builtin_inff(), l = 0.0f;
        const uint8_t* kread = lk + m32 * (2 * D);
        const int kswizzle = 16 * (hf ^ key_swizzle<D>(m32));
        const int cr = coord_of_row(m32);
        const uint8_t* vread[2];                           // of even and odd blocks of 32 coordinates
#pragma unroll
        for (int o = 0; o < 2; ++o) vread[o] = lv + 512 * hf + 16 * ((cr & 24) + ((cr & 7) ^ (4 * o + (cr >> 3))));

        load(tile0);
        for (int tile = tile0, buffer = 0; tile < end; ++tile, buffer ^= 1) {
            const uint32_t there = part.there;
            keep(buffer);
            load(tile + 1);                                // (of the tile behind the last: some page's, not used)
            __syncthreads();
            if (live) {
                float16v S[NB];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    S[b] = float16v{};
#pragma unroll
                    for (int ks = 0; ks < NKS; ++ks)
                        S[b] = wide_mfma<DT>(*reinterpret_cast<const uint4v*>(kread + buffer * C::SIDE + b * (64 * D) + ((32 * ks) ^ kswizzle)), qb[ks], S[b]);
                }
                if constexpr (POWERS) {
                    const float4v* table = reinterpret_cast<const float4v*>(powers + buffer * TT + hf * (TT / 2));
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4v times = table[4 * b + i];
#pragma unroll
                            for (int t = 0; t < 4; ++t) S[b][4 * i + t] *= times[t];
                        }
                }
                if (there != (1u << NG) - 1) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (((there >> (4 * b + e / 4)) & 1) == 0) S[b][e] = -__builtin_inff();
                }
                float top = S[0][0];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = __builtin_fmaxf(top, S[b][e]);
                top = max_xor32(top);
                if constexpr (!POWERS) top *= scale;
                // The reference moves only where a score would lead it by more than 2^4: rarely.
                const float higher = top > m + 4.0f ? top : m;
                if (__any(higher != m)) {
                    const float shrink = m == higher ? 1.0f : __builtin_amdgcn_exp2f(m - higher);
                    l *= shrink;
#pragma unroll
                    for (int ob = 0; ob < NOB; ++ob)
#pragma unroll
                        for (int e = 0; e < 16; ++e) O[ob][e] *= shrink;
                    m = higher;
                }
                const float ref = m == -__builtin_inff() ? 0.0f : m - kKvLift<PT>;
                // The weights of 16 tokens under the products of the 16 before them, whose values are read before that.
                float sum = 0.0f;
                uint4v P, rest, V[2][NOB];                 // rest: what P's rounding left
                auto weights = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float sa = S[u / 2][8 * (u & 1) + 2 * i], sb = S[u / 2][8 * (u & 1) + 2 * i + 1];
                        const float a = __builtin_amdgcn_exp2f(POWERS ? sa - ref : __builtin_fmaf(sa, scale, -ref));
                        const float b = __builtin_amdgcn_exp2f(POWERS ? sb - ref : __builtin_fmaf(sb, scale, -ref));
                        P[i] = round_pair<PT>(a, b);
                        rest[i] = round_pair<PT>(a - low_value<PT>(P[i]), b - high_value<PT>(P[i]));
                        sum += a + b;
                    }
                };
                auto read_values = [&](int u) __attribute__((always_inline)) {
#pragma unroll
                    for (int ob = 0; ob < NOB; ++ob)
                        V[u & 1][ob] = *reinterpret_cast<const uint4v*>(vread[ob & 1] + buffer * C::SIDE + (u * NOB + ob) * 1024);
                };
                read_values(0);
                weights(0);
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (u + 1 < NU) read_values(u + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int ob = 0; ob < NOB; ++ob) O[ob] = wide_mfma<PT>(V[u & 1][ob], rest, O[ob]);
#pragma unroll
                    for (int ob = 0; ob < NOB; ++ob) O[ob] = wide_mfma<PT>(V[u & 1][ob], P, O[ob]);
                    if (u + 1 < NU) weights(u + 1);
#pragma unroll
                    for (int i = 0; i < 2 * NOB; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x402, 24 / NOB, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                l += sum;
            }
        }
        l = sum_xor32(l);
        if (row < rows) {
            const int64_t at = pp.first_row + (int64_t(piece) * p.H_KV + head) * kPrefixRows + row;
#pragma unroll
            for (int ob = 0; ob < NOB; ++ob)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4v*>(p.part_o + at * D + 32 * ob + 16 * (e / 8) + 8 * hf + e % 8) =
                        float4v{O[ob][e], O[ob][e + 1], O[ob][e + 2], O[ob][e + 3]} * (F8 ? 2.0f : 1.0f);
            if (hf == 0) {
                p.part_m[at] = m;
                p.part_l[at] = l;
            }
        }
        left -= here;
        if (left <= 0) break;
        // the next group of rows
        ++piece;
        tile0 = 0;
        if (++group == groups) {
            group = 0;
            do ++prefix;
            while (prefix < p.num_prefixes && count[prefix] == 0);
            if (prefix == p.num_prefixes) break;           // (not reached: the shares end with the last tile)
        }
    }
}

// The first workgroups take the prefixes, the others what the sequences have behind them: those wait for the matrix cores, these for
// memory, so a CU has one of each (of 256 coordinates: one).
template <int D, int DT, bool F8, int HW>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_prefix_kernel(const PrefixParams pp) {
    extern __shared__ __attribute__((aligned(256))) uint8_t prefix_lds[];
    const int first = pp.shares * pp.kv.H_KV;
    if (int(blockIdx.x) < first) prefix_workgroup<D, DT, F8>(pp, int(blockIdx.x), prefix_lds);
    else kv_decode_workgroup<D, DT, F8, HW, 4 / HW, true, true>(pp.kv, int(blockIdx.x) - first, reinterpret_cast<float*>(prefix_lds));
}

// Joins the pieces of a sequence, of its own tokens and of its prefix.  A workgroup takes 4 Q neighbouring values of the G rows of one
// sequence and KV head, 256 / Q pieces at a time, each thread with a maximum and a sum of its own.
template <int D, int DT, int PT, int Q>
__global__ __launch_bounds__(256) void paged_prefix_join_kernel(const PrefixParams pp) {
    constexpr int R = 256 / Q;
    const KvDecodeParams& p = pp.kv;
    __shared__ __align__(16) float4v rows[R][Q];
    __shared__ float2v sums[R][Q];
    const int columns = p.G * D / (4 * Q);
    const int64_t unit = blockIdx.x / columns;                           // sequence and KV head
    const int seq = int(unit / p.H_KV), head = int(unit - int64_t(seq) * p.H_KV);
    const int c = 4 * (int(blockIdx.x % columns) * Q + threadIdx.x % Q), r0 = threadIdx.x / Q, h = c / D;
    int2 own = p.place[seq];
    int4 before = pp.place[seq];
    const int len = kv_length(p, seq), shared = kv_shared(p, seq, len);
    if (len <= shared) own = int2{0, 0};                                 // (of sequences without tokens nothing is written)
    if (shared == 0) before = int4{0, 0, 0, 0};
    const int pieces = own.y + before.y;
    auto row_of = [&](int i) {
        return i < own.y ? (int64_t(own.x + seq + i) * p.H_KV + head) * p.G + h
                         : pp.first_row + (int64_t(before.x + i - own.y) * p.H_KV + head) * kPrefixRows + before.z + h;
    };
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.0f;
    auto take = [&](float4v v, float m, float l) {
        const float higher = __builtin_fmaxf(top, m);
        const float a = piece_weight(top, sum, higher), b = piece_weight(m, l, higher);
        o = o * a + v * b;
        sum = sum * a + l * b;
        top = higher;
    };
    const int in_row = c - h * D;
    for (int i = r0; i < pieces; i += 4 * R) {                           // four pieces a trip
        float4v v[4];
        float m[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t row = row_of(i + k * R < pieces ? i + k * R : i);
            v[k] = *reinterpret_cast<const float4v*>(p.part_o + row * D + in_row);
            m[k] = p.part_m[row];
            l[k] = p.part_l[row];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * R < pieces) take(v[k], m[k], l[k]);
    }
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
        const int64_t out = unit * p.G;
        *reinterpret_cast<uint2v*>(p.out + out * D + c) = result_words<DT>(all * inv, p.ks != nullptr);
        if (in_row == 0 && p.lse != nullptr)
            p.lse[out + h] = den == 0.0f ? -__builtin_inff() : (highest - kKvLift<PT> + __builtin_amdgcn_logf(den)) * (1.0f / kLog2e);
    }
}

}  // namespace fq

namespace {

// How a call is divided: the sequences' own tokens as in a decode that is cut into shares, the prefixes' tiles into equal shares.
struct PrefixPlan {
    KvPlan own;
    int shares, min_tiles, members, most_pieces;
    int most_own;            // shares of the own tokens in any table
};
PrefixPlan prefix_plan(int S, int H_KV, int G, int num_prefixes, int64_t max_tokens) {
    const int64_t cus = fq_host::device_cu_count();
    PrefixPlan r;
    const int together = H_KV % 4 == 0 ? 4 : H_KV % 2 == 0 ? 2 : 1;
    auto own_shares = [&](int each) { return int((each * cus * together + H_KV - 1) / H_KV); };
    // Workgroups for the sequences' own tokens: one a CU, beside one of the prefixes', and two where the table is too narrow for much of
    // either (us, one / two: 96 sequences of 50 to 1200 tokens behind 6000 63 / 74, 64 of up to 300 behind 512 23.0 / 20.5).
    r.most_own = own_shares(2);
    r.own = {max_tokens <= 1024 ? r.most_own : own_shares(1), together, 4 / together};
    r.shares = int((cus + H_KV - 1) / H_KV);
    r.min_tiles = 2;
    r.members = fq::kPrefixRows / G;
    const int64_t groups = int64_t(S) / r.members + (num_prefixes < S ? num_prefixes : S);
    r.most_pieces = r.shares + int(groups < S ? groups : S);
    return r;
}

struct PrefixRoom {
    size_t o, m, place, prefix_place, all;
    int64_t first_row;
};
PrefixRoom prefix_room(const PrefixPlan& plan, int S, int H_Q, int H_KV, int D) {
    PrefixRoom r;
    r.first_row = (int64_t(S) + plan.most_own) * H_Q;
    const size_t rows = size_t(r.first_row) + size_t(plan.most_pieces) * size_t(H_KV) * fq::kPrefixRows;
    r.o = round_up(rows * size_t(D) * 4);
    r.m = round_up(rows * 4);
    r.place = round_up(size_t(S) * sizeof(int2));
    r.prefix_place = round_up(size_t(S) * sizeof(int4));
    r.all = r.o + 2 * r.m + r.place + r.prefix_place;
    return r;
}

template <int D, int DT, bool F8, int HW>
int launch_attend_prefix(const fq::PrefixParams& pp, const PrefixPlan& plan, hipStream_t s) {
    auto kernel = fq::paged_prefix_kernel<D, DT, F8, HW>;
    const size_t own = HW == 4 ? 0 : (size_t(4) * pp.kv.G * D + 4 * 32 + HW * 16) * 4, lds = own > fq::PrefixCfg<D>::LDS ? own : fq::PrefixCfg<D>::LDS;
    if (!fq_host::lds_limit_raised(reinterpret_cast<const void*>(kernel), lds)) return FQ_ERR_LAUNCH;
    kernel<<<unsigned(plan.shares) * unsigned(pp.kv.H_KV) + unsigned(plan.own.shares) * unsigned(pp.kv.H_KV / HW), 256, lds, s>>>(pp);
    return FQ_OK;
}

template <int D, int DT, bool F8>
int launch_prefix(const fq::PrefixParams& pp, const PrefixPlan& plan, hipStream_t s) {
    constexpr int PT = F8 ? FQ_BF16 : DT;
    const int st = plan.own.heads == 4 ? launch_attend_prefix<D, DT, F8, 4>(pp, plan, s)
                   : plan.own.heads == 2 ? launch_attend_prefix<D, DT, F8, 2>(pp, plan, s) : launch_attend_prefix<D, DT, F8, 1>(pp, plan, s);
    if (st != FQ_OK) return st;
    // As many values a workgroup as leave enough workgroups: then a thread has its values' pieces to itself, and the trips to memory that every
    // workgroup begins with are fewer
    const int64_t values = int64_t(pp.kv.S) * pp.kv.H_KV * pp.kv.G * D, enough = 2 * int64_t(fq_host::device_cu_count());
    auto fits = [&](int per) { return pp.kv.G * D % per == 0 && values / per >= enough; };
    if (fits(1024)) fq::paged_prefix_join_kernel<D, DT, PT, 256><<<unsigned(values / 1024), 256, 0, s>>>(pp);
    else if (fits(512)) fq::paged_prefix_join_kernel<D, DT, PT, 128><<<unsigned(values / 512), 256, 0, s>>>(pp);
    else if (fits(256)) fq::paged_prefix_join_kernel<D, DT, PT, 64><<<unsigned(values / 256), 256, 0, s>>>(pp);
    else fq::paged_prefix_join_kernel<D, DT, PT, 16><<<unsigned(values / 64), 256, 0, s>>>(pp);
    return fq_host::check_launch();
}

template <int D>
int launch_prefix_type(const fq::PrefixParams& pp, const PrefixPlan& plan, bool f8, int dtype, hipStream_t s) {
    if (dtype == FQ_BF16) return f8 ? launch_prefix<D, FQ_BF16, true>(pp, plan, s) : launch_prefix<D, FQ_BF16, false>(pp, plan, s);
    return f8 ? launch_prefix<D, FQ_F16, true>(pp, plan, s) : launch_prefix<D, FQ_F16, false>(pp, plan, s);
}

}  // namespace

extern "C" size_t fq_paged_prefix_decode_workspace_bytes(int num_seqs, int H_Q, int H_KV, int D, int num_prefixes) {
    if (check_kv_shape(num_seqs, H_Q, H_KV, D, 16, 1, 1) != FQ_OK || num_seqs == 0 || num_prefixes < 0 || num_prefixes > fq::kPrefixMost) return 0;
    return prefix_room(prefix_plan(num_seqs, H_KV, H_Q / H_KV, num_prefixes, 0), num_seqs, H_Q, H_KV, D).all;
}

extern "C" int fq_paged_prefix_decode(const void* q, const int64_t* q_strides, const void* key_cache, const int64_t* key_strides,
                                      const void* value_cache, const int64_t* value_strides, const uint8_t* key_scales,
                                      const int64_t* key_scale_strides, const uint8_t* value_scales, const int64_t* value_scale_strides,
                                      const int32_t* block_table, int64_t block_table_stride, const int32_t* seq_lens,
                                      const int32_t* prefix_ids, const int32_t* prefix_lens, int num_prefixes, void* out, float* lse,
                                      int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq, int64_t num_blocks,
                                      float sm_scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, num_blocks);
    if (bad != FQ_OK) return bad;
    if (dtype != FQ_F16 && dtype != FQ_BF16) return FQ_ERR_UNSUPPORTED_DTYPE;
    if (block_table_stride < 0 || num_prefixes < 0 || num_prefixes > fq::kPrefixMost) return FQ_ERR_BAD_SHAPE;
    if (num_seqs == 0) return FQ_OK;
    const bool f8 = key_scales != nullptr || value_scales != nullptr;
    if (!q || !q_strides || !key_cache || !key_strides || !value_cache || !value_strides || !block_table || !seq_lens || !prefix_ids || !out ||
        (num_prefixes > 0 && !prefix_lens) || !workspace ||
        (f8 && (!key_scales || !key_scale_strides || !value_scales || !value_scale_strides)))
        return FQ_ERR_NULL_POINTER;
    const int unit = f8 ? 16 : 8;
    for (int i = 0; i < 3; ++i)
        if (key_strides[i] % unit != 0 || value_strides[i] % unit != 0 || (i < 2 && q_strides[i] % 8 != 0)) return FQ_ERR_MISALIGNED;
    if (!fq_host::aligned(q, 16) || !fq_host::aligned(key_cache, 16) || !fq_host::aligned(value_cache, 16) || !fq_host::aligned(out, 16) ||
        (f8 && !(codes_aligned(key_cache, key_strides, key_scales, key_scale_strides) &&
                 codes_aligned(value_cache, value_strides, value_scales, value_scale_strides))))
        return FQ_ERR_MISALIGNED;
    const PrefixPlan plan = prefix_plan(num_seqs, H_KV, H_Q / H_KV, num_prefixes, int64_t(max_blocks_per_seq) * block_size);
    const PrefixRoom room = prefix_room(plan, num_seqs, H_Q, H_KV, D);
    // (units of work are counted in 32 bits)
    const int64_t max_tokens = int64_t(max_blocks_per_seq) * block_size;
    if (max_tokens > 0x7fff0000LL) return FQ_ERR_BAD_SHAPE;          // tiles are asked for ahead
    const int between = plan.own.waves * (f8 ? 2 : 1);
    if (int64_t(num_seqs) * ((max_tokens + fq::kKvTile - 1) / fq::kKvTile + between) > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    if ((int64_t(num_seqs) / plan.members + num_prefixes) * (max_tokens / (8192 / D) + 1) > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    if (room.o / (size_t(D) * 4) * size_t(D / 32) > size_t(0x7fffffff)) return FQ_ERR_BAD_SHAPE;
    if (workspace_bytes < room.all) return FQ_ERR_WORKSPACE;
    if (!fq_host::aligned(workspace, 256)) return FQ_ERR_MISALIGNED;
    fq::PrefixParams pp = {};
    fq::KvDecodeParams& p = pp.kv;
    set_up_params(p, q, q_strides, block_table, block_table_stride, seq_lens, out, lse, num_seqs, H_Q, H_KV, block_size, max_blocks_per_seq,
                  num_blocks, sm_scale, 0, plan.own);
    char* ws = static_cast<char*>(workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_m = reinterpret_cast<float*>(ws + room.o);
    p.part_l = reinterpret_cast<float*>(ws + room.o + room.m);
    p.place = reinterpret_cast<int2*>(ws + room.o + 2 * room.m);
    pp.place = reinterpret_cast<int4*>(ws + room.o + 2 * room.m + room.place);
    p.between = between;
    p.prefix_ids = prefix_ids;
    p.prefix_lens = prefix_lens;
    p.num_prefixes = num_prefixes;
    pp.first_row = room.first_row;
    pp.shares = plan.shares;
    pp.min_tiles = plan.min_tiles;
    pp.members = plan.members;
    if (f8) {
        set_codes(p, static_cast<const uint8_t*>(key_cache), key_strides, static_cast<const uint8_t*>(value_cache), value_strides, key_scales,
                  key_scale_strides, value_scales, value_scale_strides);
    } else {
        set_rows(p, key_cache, key_strides, value_cache, value_strides);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_prefix_type<64>(pp, plan, f8, dtype, s);
        case 128: return launch_prefix_type<128>(pp, plan, f8, dtype, s);
        default: return launch_prefix_type<256>(pp, plan, f8, dtype, s);
    }
}
