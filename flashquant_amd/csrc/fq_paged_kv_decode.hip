// Attention of one new token per sequence over a paged cache of 16-bit keys and values.
//
//   o_h = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q_h . k_j - m),  c = sm_scale log2(e),  m = max_j c q_h . k_j
//
// over the tokens j of the sequence (with a window: the last ones); the G = H_Q / H_KV query heads of a KV head share its rows.
//
// What bounds it: every key and value is read once, 4 D bytes a token and KV head for 4 G D flops, so HBM does.  The tile loop
// therefore only has to keep enough loads in flight, and is laid out so that nothing but registers stands between a load and
// the matrix cores:
//   * A wavefront takes 32 keys at a time.  S^T = K Q^T runs on v_mfma_f32_16x16x32: the A operand is a key's row as it lies in
//     memory (16 bytes a lane).  Row m of tile t is key 8 (m / 4) + 4 t + m % 4, so that after two tiles lane (g, h) holds the
//     scores of keys 8 g .. 8 g + 7 for head h: exactly the B operand of O^T = V^T P, without a move between lanes.
//   * A lane loads coordinates 8 n .. 8 n + 7 of the values of keys 8 g .. 8 g + 7 (whole rows of 256 bytes a group of 16
//     lanes) and turns them into the A operand, 8 keys of one coordinate, with half a v_perm_b32 an element.
//   * O^T has the head along the lanes: the running maximum, sum and rescaling are a lane's own.
//   * A weight goes to the second product as two 16-bit terms (16 significant bits and more), so that the only rounding
//     that shows is that of the output; the matrix cores are idle otherwise.  Maximum and sum are float32, of the unrounded
//     weights.
// The wavefronts of a workgroup take a part's tiles in turn and are joined in LDS.  Long sequences are cut into parts, joined by
// a second launch (find_part below).
#include "fq_device.hpp"

namespace fq {

constexpr int kKvTile = 32;               // keys of a wavefront's step
constexpr float kKvLift = 10.0f;          // weights are kept times 2^10: their second terms stay normal in fp16

struct KvDecodeParams {
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int32_t* table;
    const int32_t* lens;
    uint16_t* out;
    float* lse;                           // may be null
    float* part_o;                        // (S + extra, H_KV, G, D)
    float* part_m;                        // (S + extra, H_KV, G)
    float* part_l;
    int64_t q_seq, q_head;                // strides in elements
    int64_t k_block, k_token, k_head, v_block, v_token, v_head;
    int64_t table_row;
    int S, H_KV, G, page_log2, max_blocks, num_blocks, window;
    int extra;                            // parts beyond one a sequence, of a KV head; 0: no sequence is cut
    int min_tiles;                        // of a part of a sequence that is cut
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

// Which part of which sequence is number x.  Nothing on the host knows the lengths, so every workgroup works it out from them:
// a part has `size` tiles, so chosen that all sequences together have at most S + extra parts; each sequence is then cut into
// equal ones.  Arithmetic on the lengths alone: the same in every workgroup and in the launch that joins the parts.
struct KvPart {
    int seq, part, parts, base;           // base: number of the sequence's first part
    KvSpan span;
};
__device__ __forceinline__ int kv_part_size(const KvDecodeParams& p, int lane) {
    uint32_t total = 0;
    for (int s = 0; s < p.S; s += kWave) total += uint32_t(s + lane < p.S ? kv_span(p, p.lens[s + lane]).tiles : 0);
    total = wave_sum(total);
    const int share = int((total + uint32_t(p.extra) - 1) / uint32_t(p.extra));
    return share > p.min_tiles ? share : p.min_tiles;
}
__device__ __forceinline__ int kv_parts(int tiles, int size) { return tiles <= size ? 1 : (tiles + size - 1) / size; }

// by_seq: x is a sequence and the answer its first part; else x is a part's number.  False: there is none of that number.
template <bool by_seq>
__device__ __forceinline__ bool find_part(const KvDecodeParams& p, int x, int lane, KvPart& r) {
    if (p.extra == 0) {
        r = {x, 0, 1, x, kv_span(p, p.lens[x])};
        return true;
    }
    const int size = kv_part_size(p, lane);
    int before = 0;
    for (int s = 0; s < p.S; s += kWave) {
        const int len = s + lane < p.S ? p.lens[s + lane] : 0;
        const int n = s + lane < p.S ? kv_parts(kv_span(p, len).tiles, size) : 0;
        int upto = n;                                        // inclusive sum over the lanes
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int below = __shfl_up(upto, d, kWave);
            upto += lane >= d ? below : 0;
        }
        const int all = __builtin_amdgcn_readlane(upto, kWave - 1);
        const bool here = by_seq ? x < s + kWave : x < before + all;
        if (here) {
            const int at = by_seq ? x - s : __ffsll(static_cast<unsigned long long>(__ballot(before + upto > x))) - 1;
            const int l = __builtin_amdgcn_readlane(len, at);
            r.seq = s + at;
            r.parts = __builtin_amdgcn_readlane(n, at);
            r.base = before + __builtin_amdgcn_readlane(upto, at) - r.parts;
            r.part = by_seq ? 0 : x - r.base;
            r.span = kv_span(p, l);
            return true;
        }
        before += all;
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

// Words of a lane's piece of one value row: 8 coordinates of 128, 4 of 64.
template <int D> struct ValueWords { static constexpr int n = D == 64 ? 2 : 4; };

template <int D, int DT, int W>
__global__ __launch_bounds__(W * kWave) void paged_kv_decode_kernel(const KvDecodeParams p) {
    constexpr int KJ = D / 32;                       // steps of 32 coordinates in a score
    constexpr int VH = D == 256 ? 2 : 1;             // halves of 128 coordinates
    constexpr int VW = ValueWords<D>::n;
    constexpr int VE = 2 * VW;                       // coordinates of a lane's piece
    extern __shared__ __align__(16) float lds[];     // (W, G, D), then (W, 2, 16), then (2, 16)
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n = lane & 15, g = lane >> 4;
    const int G = p.G;
    const int x = blockIdx.x / p.H_KV, head = blockIdx.x - x * p.H_KV;

    KvPart at;
    if (!find_part<false>(p, x, lane, at)) return;
    int begin = 0, end = at.span.tiles;
    if (at.parts > 1) {
        const int each = at.span.tiles / at.parts, more = at.span.tiles - each * at.parts;
        begin = at.part * each + (at.part < more ? at.part : more);
        end = begin + each + (at.part < more ? 1 : 0);
    }
    begin += at.span.first;
    end += at.span.first;

    const int32_t* table = p.table + int64_t(at.seq) * p.table_row;
    const uint16_t* kbase = p.kc + head * p.k_head + 8 * g + int64_t(n & 3) * p.k_token;
    const uint16_t* vbase = p.vc + head * p.v_head + VE * n;
    const int page_mask = (1 << p.page_log2) - 1;

    // the block of the 8 keys that this lane reads a key of, and of those that it reads the values of
    auto block_of = [&](int tile, int group) {
        const int b = (tile * kKvTile + 8 * group) >> p.page_log2;
        return table[b < p.max_blocks ? b : p.max_blocks - 1];
    };
    auto in_cache = [&](int block) { return uint32_t(block) < uint32_t(p.num_blocks); };

    uint4v kr[2][KJ];
    uint32_t vr[8][VH][VW];
    auto load_keys = [&](int tile, int block) {
        const int group = n >> 2;
        const uint16_t* src = kbase + int64_t(in_cache(block) ? block : 0) * p.k_block +
                              int64_t((tile * kKvTile + 8 * group) & page_mask) * p.k_token;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int j = 0; j < KJ; ++j) kr[t][j] = *reinterpret_cast<const uint4v*>(src + 32 * j);
            src += 4 * p.k_token;
        }
    };
    auto load_values = [&](int tile, int block) {
        const uint16_t* src = vbase + int64_t(in_cache(block) ? block : 0) * p.v_block +
                              int64_t((tile * kKvTile + 8 * g) & page_mask) * p.v_token;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int h = 0; h < VH; ++h) {
                if constexpr (VW == 4) {
                    const uint4v w = *reinterpret_cast<const uint4v*>(src + 128 * h);
                    vr[i][h][0] = w.x; vr[i][h][1] = w.y; vr[i][h][2] = w.z; vr[i][h][3] = w.w;
                } else {
                    const uint2v w = *reinterpret_cast<const uint2v*>(src);
                    vr[i][h][0] = w.x; vr[i][h][1] = w.y;
                }
            }
            src += p.v_token;
        }
    };

    float4v acc[VH][VE];
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[h][e] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.0f;

    int tile = begin + wave;
    if (tile < end) {
        int kblock = block_of(tile, n >> 2), vblock = block_of(tile, g);
        load_keys(tile, kblock);
        load_values(tile, vblock);
        uint4v qr[KJ];
        {
            const uint16_t* src = p.q + int64_t(at.seq) * p.q_seq + int64_t(head * G + (n < G ? n : 0)) * p.q_head + 8 * g;
#pragma unroll
            for (int j = 0; j < KJ; ++j) qr[j] = n < G ? *reinterpret_cast<const uint4v*>(src + 32 * j) : uint4v{0u, 0u, 0u, 0u};
        }
        int next_k = 0, next_v = 0;
        if (tile + W < end) { next_k = block_of(tile + W, n >> 2); next_v = block_of(tile + W, g); }
        for (; tile < end; tile += W) {
            const bool more = tile + W < end;
            float4v s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[t] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KJ; ++j) s[t] = kv_mfma<DT>(kr[t][j], qr[j], s[t]);
            }
            __builtin_amdgcn_sched_barrier(0);
            int after_k = 0, after_v = 0;
            if (more) {
                load_keys(tile + W, next_k);
                if (tile + 2 * W < end) { after_k = block_of(tile + 2 * W, n >> 2); after_v = block_of(tile + 2 * W, g); }
            }
            __builtin_amdgcn_sched_barrier(0);
            float sv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) sv[i] = s[i >> 2][i & 3] * p.scale_log2;
            // whole tiles whose pages are all in the cache need no mask
            const int key = tile * kKvTile + 8 * g;
            const bool page_ok = in_cache(vblock);
            const bool whole = tile * kKvTile >= at.span.lo && tile * kKvTile + kKvTile <= at.span.len && __all(page_ok);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool seen = page_ok && key + i >= at.span.lo && key + i < at.span.len;
                    sv[i] = seen ? sv[i] : -__builtin_inff();
                }
            }
            float top = sv[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, sv[i]);
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
            const float ref = m == -__builtin_inff() ? 0.0f : m - kKvLift;
            uint4v hi, lo;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float a = __builtin_amdgcn_exp2f(sv[i] - ref), b = __builtin_amdgcn_exp2f(sv[i + 1] - ref);
                l += a + b;
                hi[i / 2] = round_pair<DT>(a, b);
                lo[i / 2] = round_pair<DT>(a - low_value<DT>(hi[i / 2]), b - high_value<DT>(hi[i / 2]));
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool seen = page_ok && key + i >= at.span.lo && key + i < at.span.len;
#pragma unroll
                    for (int h = 0; h < VH; ++h)
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[i][h][w] = seen ? vr[i][h][w] : 0u;
                }
            }
            uint4v vt[VH][VE];
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int e = 0; e < VE; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vt[h][e][i] = __builtin_amdgcn_perm(vr[2 * i + 1][h][e / 2], vr[2 * i][h][e / 2],
                                                            e & 1 ? 0x07060302u : 0x05040100u);
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_values(tile + W, next_v);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < VH; ++h)
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    acc[h][e] = kv_mfma<DT>(vt[h][e], lo, acc[h][e]);
                    acc[h][e] = kv_mfma<DT>(vt[h][e], hi, acc[h][e]);
                }
            kblock = next_k; vblock = next_v;
            next_k = after_k; next_v = after_v;
        }
        l = sum_xor32(sum_xor16(l));
    }

    // the wavefronts' results, joined: lane (g, h) holds coordinates VE (4 g + r) + e of head h
    float* sm = lds + W * G * D;
    float* total = sm + W * 32;
    if (g == 0) {
        sm[wave * 32 + n] = m;
        sm[wave * 32 + 16 + n] = l;
    }
    __syncthreads();
    float top = sm[n];
#pragma unroll
    for (int w = 1; w < W; ++w) top = __builtin_fmaxf(top, sm[w * 32 + n]);
    if (wave == 0 && g == 0) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float mw = sm[w * 32 + n], lw = sm[w * 32 + 16 + n];
            sum += lw * piece_weight(mw, lw, top);
        }
        total[n] = top;
        total[16 + n] = sum;
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
    const int64_t row = int64_t(x) * p.H_KV + head;                  // of the parts
    const int64_t orow = (int64_t(at.seq) * p.H_KV + head) * G;      // of the outputs
    for (int i = 4 * int(threadIdx.x); i < G * D; i += 4 * W * kWave) {
        float4v o = *reinterpret_cast<const float4v*>(lds + i);
#pragma unroll
        for (int w = 1; w < W; ++w) o += *reinterpret_cast<const float4v*>(lds + w * G * D + i);
        if (at.parts == 1) {
            const float inv = inverse_sum(total[16 + i / D]);
            *reinterpret_cast<uint2v*>(p.out + orow * D + i) = uint2v{round_pair<DT>(o.x * inv, o.y * inv), round_pair<DT>(o.z * inv, o.w * inv)};
        } else {
            *reinterpret_cast<float4v*>(p.part_o + row * G * D + i) = o;
        }
    }
    if (int(threadIdx.x) < G) {
        const float mt = total[threadIdx.x], lt = total[16 + threadIdx.x];
        if (at.parts > 1) {
            p.part_m[row * G + threadIdx.x] = mt;
            p.part_l[row * G + threadIdx.x] = lt;
        } else if (p.lse != nullptr) {
            p.lse[orow + threadIdx.x] = lt == 0.0f ? -__builtin_inff() : (mt - kKvLift + __builtin_amdgcn_logf(lt)) * (1.0f / kLog2e);
        }
    }
}

// Joins the parts of the sequences that have several; one workgroup a sequence and query head.
template <int D, int DT>
__global__ __launch_bounds__(256) void paged_kv_join_kernel(const KvDecodeParams p) {
    constexpr int Q = D / 4;                         // lanes of a row
    constexpr int R = 256 / Q;                       // rows at a time
    __shared__ __align__(16) float rows[R][D];
    __shared__ float wave_m[4], sums[R];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int H_Q = p.H_KV * p.G;
    const int seq = blockIdx.x / H_Q, hq = blockIdx.x - seq * H_Q;
    KvPart at;
    find_part<true>(p, seq, lane, at);
    if (at.parts == 1) return;
    // parts of one KV head lie H_KV * G rows apart
    const int64_t first = int64_t(at.base) * H_Q + hq;
    float top = -__builtin_inff();
    for (int i = threadIdx.x; i < at.parts; i += 256) top = __builtin_fmaxf(top, p.part_m[first + int64_t(i) * H_Q]);
    top = wave_max(top);
    if (lane == 0) wave_m[wave] = top;
    __syncthreads();
    top = __builtin_fmaxf(__builtin_fmaxf(wave_m[0], wave_m[1]), __builtin_fmaxf(wave_m[2], wave_m[3]));
    const int c = 4 * (threadIdx.x % Q), r0 = threadIdx.x / Q;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.0f;
    for (int i = r0; i < at.parts; i += R) {
        const int64_t row = first + int64_t(i) * H_Q;
        const float l = p.part_l[row], w = piece_weight(p.part_m[row], l, top);
        o += *reinterpret_cast<const float4v*>(p.part_o + row * D + c) * w;
        sum += l * w;
    }
    *reinterpret_cast<float4v*>(&rows[r0][c]) = o;
    if (threadIdx.x % Q == 0) sums[r0] = sum;
    __syncthreads();
    if (threadIdx.x < Q) {
        float den = sums[0];
        for (int r = 1; r < R; ++r) {
            o += *reinterpret_cast<const float4v*>(&rows[r][c]);
            den += sums[r];
        }
        const float inv = inverse_sum(den);
        const int64_t out = int64_t(seq) * H_Q + hq;
        *reinterpret_cast<uint2v*>(p.out + out * D + c) = uint2v{round_pair<DT>(o.x * inv, o.y * inv), round_pair<DT>(o.z * inv, o.w * inv)};
        if (threadIdx.x == 0 && p.lse != nullptr)
            p.lse[out] = den == 0.0f ? -__builtin_inff() : (top - kKvLift + __builtin_amdgcn_logf(den)) * (1.0f / kLog2e);
    }
}

}  // namespace fq

namespace {

constexpr int kWaves = 8;

// Parts beyond one a sequence, of a KV head (0: no sequence is cut, and no second launch).
int kv_extra(int S, int H_KV, int64_t max_tokens) {
    const int64_t tiles = (max_tokens + fq::kKvTile - 1) / fq::kKvTile;
    if (tiles <= 2 * kWaves || int64_t(S) * tiles >= (1LL << 31)) return 0;
    const int target = 2 * fq_host::device_cu_count();
    return (target + H_KV - 1) / H_KV;
}

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
    size_t o, m, all;
};
KvRoom kv_room(int S, int H_Q, int D, int extra) {
    const size_t rows = (size_t(S) + size_t(extra)) * size_t(H_Q);
    KvRoom r;
    r.o = round_up(rows * size_t(D) * 4);
    r.m = round_up(rows * 4);
    r.all = extra == 0 ? 0 : r.o + 2 * r.m;
    return r;
}

template <int D, int DT>
int launch_kv(const fq::KvDecodeParams& p, hipStream_t s) {
    constexpr int W = D == 256 ? 4 : kWaves;
    const size_t lds = (size_t(W) * p.G * D + W * 32 + 32) * 4;
    auto kernel = fq::paged_kv_decode_kernel<D, DT, W>;
    if (lds > 32768 && !fq_host::lds_limit_raised(reinterpret_cast<const void*>(kernel), lds)) return FQ_ERR_LAUNCH;
    kernel<<<unsigned(p.S + p.extra) * unsigned(p.H_KV), W * 64, lds, s>>>(p);
    if (p.extra > 0) fq::paged_kv_join_kernel<D, DT><<<unsigned(p.S) * unsigned(p.H_KV * p.G), 256, 0, s>>>(p);
    return fq_host::check_launch();
}

template <int D>
int launch_kv_type(const fq::KvDecodeParams& p, int dtype, hipStream_t s) {
    return dtype == FQ_BF16 ? launch_kv<D, FQ_BF16>(p, s) : launch_kv<D, FQ_F16>(p, s);
}

}  // namespace

extern "C" size_t fq_paged_kv_decode_workspace_bytes(int num_seqs, int H_Q, int H_KV, int D, int block_size, int max_blocks_per_seq) {
    if (check_kv_shape(num_seqs, H_Q, H_KV, D, block_size, max_blocks_per_seq, 1) != FQ_OK || num_seqs == 0) return 0;
    const int extra = kv_extra(num_seqs, H_KV, int64_t(max_blocks_per_seq) * block_size);
    return kv_room(num_seqs, H_Q, D, extra).all;
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
    const int extra = kv_extra(num_seqs, H_KV, int64_t(max_blocks_per_seq) * block_size);
    if ((int64_t(num_seqs) + extra) * H_Q > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    const KvRoom room = kv_room(num_seqs, H_Q, D, extra);
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
    p.q_seq = q_strides[0]; p.q_head = q_strides[1];
    p.k_block = key_strides[0]; p.k_token = key_strides[1]; p.k_head = key_strides[2];
    p.v_block = value_strides[0]; p.v_token = value_strides[1]; p.v_head = value_strides[2];
    p.table_row = block_table_stride;
    p.S = num_seqs; p.H_KV = H_KV; p.G = H_Q / H_KV;
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.max_blocks = max_blocks_per_seq; p.num_blocks = int(num_blocks); p.window = window;
    p.extra = extra; p.min_tiles = kWaves;
    p.scale_log2 = sm_scale * fq::kLog2e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (D) {
        case 64: return launch_kv_type<64>(p, dtype, s);
        case 128: return launch_kv_type<128>(p, dtype, s);
        default: return launch_kv_type<256>(p, dtype, s);
    }
}
