// Pages, slots and positions of a step's new tokens, from the requests' lengths: the inputs of every paged entry point, made on
// the GPU.
//
// Request r holds context_r tokens and brings query_r new ones.  Its pages are the first ceil(context / B) entries of its row of the
// block table; a page that its new tokens begin is taken from the list of free ones, in the order of requests and tokens:
//   new_r = ceil((context_r + query_r) / B) - ceil(context_r / B),  page i of them = free[start + sum_{s < r} new_s + i].
// What bounds it: nothing but latency (16 bytes a token; lengths, then free pages or the block table, then the stores: three trips
// to memory).  So it is one launch of independent workgroups: each adds up all lengths for itself, keeps the requests that reach
// into its 256 tokens in LDS, and a thread then finds the request of its token as the last one that begins at or before it.
// A new page has a first token, which is new too: its thread writes the page into the block table.  What a thread reads there are
// pages from before, so nothing that one workgroup writes is read by another.
#include "fq_common.hpp"

namespace fq {

constexpr int kScheduleThreads = 256;
constexpr int kScheduleMost = 8;

struct ScheduleParams {
    const int32_t* context;
    const int32_t* query;
    int32_t* table;
    const int32_t* free_blocks;
    const int32_t* free_start;      // may be null: 0
    int32_t* free_end;
    int64_t* slots;
    int64_t* positions;
    int32_t* seq_lens;
    int32_t* cu;
    int64_t table_row;
    int64_t num_tokens;
    int S, max_blocks, num_free, page_log2;
    int capped;                     // tokens beyond num_tokens do not count
};

// inclusive sums over the workgroup of two values; `sum` gets those of all threads
__device__ __forceinline__ int2 sums_upto(int2 v, int2 (&waves)[kScheduleThreads / kWave], int2& sum) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int x = __shfl_up(v.x, d, kWave), y = __shfl_up(v.y, d, kWave);
        v.x += lane >= d ? x : 0;
        v.y += lane >= d ? y : 0;
    }
    __syncthreads();                // the sums of the time before have been read
    if (lane == kWave - 1) waves[wave] = v;
    __syncthreads();
    sum = int2{0, 0};
#pragma unroll
    for (int w = 0; w < kScheduleThreads / kWave; ++w) {
        if (w < wave) { v.x += waves[w].x; v.y += waves[w].y; }
        sum.x += waves[w].x;
        sum.y += waves[w].y;
    }
    return v;
}

// MOST: requests of a thread at a time, added up before the workgroup adds up
template <int MOST>
__global__ __launch_bounds__(kScheduleThreads) void paged_schedule_kernel(const ScheduleParams p) {
    __shared__ int2 waves[kScheduleThreads / kWave];
    __shared__ int owner[kScheduleThreads], owner_cu[kScheduleThreads], owner_context[kScheduleThreads], owner_page[kScheduleThreads];
    __shared__ int wave_last[kScheduleThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t lo = int64_t(blockIdx.x) * kScheduleThreads, hi = lo + kScheduleThreads;
    const int page = 1 << p.page_log2;
    const int64_t room = int64_t(p.max_blocks) << p.page_log2;
    owner[tid] = -1;
    const int start = p.free_start != nullptr ? p.free_start[0] : 0;
    int2 before = {0, 0};           // tokens and pages of the requests so far
    int each = (p.S + kScheduleThreads - 1) / kScheduleThreads;
    each = MOST == 1 || each < 1 ? 1 : each < MOST ? each : MOST;
    for (int s = 0; s < p.S; s += each * kScheduleThreads) {
        int context[MOST], query[MOST];
        const int r0 = s + tid * each;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const bool mine = i < each && r0 + i < p.S;
            context[i] = mine ? p.context[r0 + i] : 0;
            query[i] = mine ? p.query[r0 + i] : 0;
        }
        auto pages_of = [&](int i, int64_t& has) {           // new ones; `has`: tokens after the step
            const int64_t had = context[i] < room ? context[i] : room;
            has = int64_t(context[i]) + query[i];
            if (has > room) has = room;
            return int((has + page - 1) >> p.page_log2) - int((had + page - 1) >> p.page_log2);
        };
        int2 mine = {0, 0};
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            context[i] = context[i] > 0 ? context[i] : 0;
            query[i] = query[i] > 0 ? query[i] : 0;
            int64_t has;
            mine.x += query[i];
            mine.y += pages_of(i, has);
        }
        int2 all;
        int2 at = sums_upto(mine, waves, all);               // (its barriers also lie between the clearing of `owner` and what follows)
        at = int2{before.x + at.x - mine.x, before.y + at.y - mine.y};
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            if (i >= each || r0 + i >= p.S) break;
            int64_t has;
            int pages = pages_of(i, has);
            if (query[i] > 0 && at.x < hi && int64_t(at.x) + query[i] > lo) {      // of the tokens [lo, hi)
                const int o = int(at.x > lo ? at.x - lo : 0);
                owner[o] = r0 + i;
                owner_cu[o] = at.x;
                owner_context[o] = context[i];
                owner_page[o] = at.y;
            }
            const int64_t left = p.num_tokens - at.x;                              // room for this request's tokens
            at.x += query[i];
            if (p.capped && left < query[i]) {
                // only tokens with room take the pages that they begin (those of all requests before this one do)
                query[i] = left > 0 ? int(left) : 0;
                pages = pages_of(i, has);
            }
            at.y += pages;
            if (blockIdx.x == 0) {
                p.seq_lens[r0 + i] = int(has);
                p.cu[r0 + i + 1] = p.capped && at.x > p.num_tokens ? int(p.num_tokens) : at.x;
                // the request of the last token with room takes the last page
                if (p.capped && left > 0 && at.x >= p.num_tokens && query[i] > 0) p.free_end[0] = start + at.y;
            }
        }
        before.x += all.x;
        before.y += all.y;
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.cu[0] = 0;
        if (!p.capped || before.x < p.num_tokens) p.free_end[0] = start + before.y;
        else if (p.num_tokens == 0) p.free_end[0] = start;
    }
    __syncthreads();
    // the last request that begins at or before this thread's token
    const uint64_t begins = __ballot(owner[tid] >= 0);
    if (lane == 0) wave_last[wave] = begins != 0 ? wave * kWave + 63 - __clzll(static_cast<long long>(begins)) : -1;
    __syncthreads();
    const int64_t token = lo + tid;
    if (token >= p.num_tokens) return;
    const uint64_t mine = begins & (~uint64_t(0) >> (63 - lane));
    int at = mine != 0 ? wave * kWave + 63 - __clzll(static_cast<long long>(mine)) : -1;
    for (int w = wave - 1; at < 0 && w >= 0; --w) at = wave_last[w];
    if (token >= before.x || at < 0) {                       // behind the last new token
        p.slots[token] = -1;
        p.positions[token] = 0;
        return;
    }
    const int context = owner_context[at];
    const int64_t position = context + (token - owner_cu[at]);
    int64_t slot = -1;
    if (position < room) {
        const int b = int(position >> p.page_log2), in_page = int(position & (page - 1));
        const int held = int((int64_t(context) + page - 1) >> p.page_log2);
        int32_t* entry = p.table + int64_t(owner[at]) * p.table_row + b;
        int block;
        if (b < held) {
            block = *entry;
        } else {
            const int64_t i = int64_t(start) + owner_page[at] + (b - held);
            block = i >= 0 && i < p.num_free ? p.free_blocks[i] : -1;
            if (in_page == 0) *entry = block;
        }
        if (block >= 0) slot = (int64_t(block) << p.page_log2) + in_page;
    }
    p.slots[token] = slot;
    p.positions[token] = position;
}

// What follows a schedule, in one launch: lengths and first free page as the next one finds them, and a row of pages and a length
// for each of the step's tokens.  A schedule packs the tokens and leaves out requests that bring none, so token i is not of request
// i: attention of single tokens goes by these rows.
//   What bounds it: latency, and for wide tables the copy.  A workgroup takes up to 2048 entries of one row.  It finds the request with
// one look at all of `cu`, a trip to memory for every 1024 requests, where a search would take one for every halving.  Measured: 64 tokens
// of 256 pages 3.3 us, of 8192 4.0, 512 of 8192 (34 MB) 6.9 (4.9 TB/s); a whole schedule of 64 sequences in a graph 8.0, and 8.7 with two
// launches that moved lengths and first page alone.
constexpr int kRowEntries = 8 * kScheduleThreads;

struct AdvanceParams {
    const int32_t* seq_lens;
    const int32_t* free_end;
    int32_t* context;
    int32_t* free_start;
    const int32_t* cu;
    const int64_t* positions;
    const int32_t* table;
    int32_t* token_table;           // (num_tokens, max_blocks)
    int32_t* token_lens;
    const int32_t* prefix_ids;      // of every request, with shared prefixes; else null
    int32_t* token_prefix;
    int64_t table_row;
    int S, max_blocks, num_blocks, page_log2;
    int state_groups, parts;        // workgroups of the state, those of a token's row
};

__global__ __launch_bounds__(kScheduleThreads) void paged_advance_kernel(const AdvanceParams p) {
    const int tid = threadIdx.x;
    if (int(blockIdx.x) < p.state_groups) {
        const int r = int(blockIdx.x) * kScheduleThreads + tid;
        if (r < p.S) p.context[r] = p.seq_lens[r];
        if (r == 0) {
            const int end = p.free_end[0];
            p.free_start[0] = end < p.num_blocks ? end : p.num_blocks;
        }
        return;
    }
    __shared__ int owner;
    if (tid == 0) owner = -1;
    __syncthreads();
    const int token = (int(blockIdx.x) - p.state_groups) / p.parts, part = (int(blockIdx.x) - p.state_groups) % p.parts;
#pragma unroll 4
    for (int s = tid; s < p.S; s += kScheduleThreads)
        if (p.cu[s] <= token && token < p.cu[s + 1]) owner = s;          // of one request at most
    __syncthreads();
    const int s = owner;                                                 // none behind the last token: nothing is seen
    if (part == 0 && tid == 0) {
        const int64_t room = int64_t(p.max_blocks) << p.page_log2, upto = p.positions[token] + 1;
        p.token_lens[token] = s < 0 ? 0 : int(upto < room ? upto : room);
        if (p.token_prefix != nullptr) p.token_prefix[token] = s < 0 ? -1 : p.prefix_ids[s];
    }
    const int32_t* from = p.table + int64_t(s < 0 ? 0 : s) * p.table_row;
    int32_t* to = p.token_table + int64_t(token) * p.max_blocks;
#pragma unroll
    for (int k = 0; k < kRowEntries / kScheduleThreads; ++k) {
        const int i = part * kRowEntries + k * kScheduleThreads + tid;
        if (i < p.max_blocks) to[i] = s < 0 ? -1 : from[i];
    }
}

}  // namespace fq

namespace {

int schedule(const int32_t* context_lens, const int32_t* query_lens, int32_t* block_table, int64_t block_table_stride, const int32_t* free_blocks,
             int64_t num_free, const int32_t* free_start, int32_t* free_end, int64_t* slot_mapping, int64_t* positions, int32_t* seq_lens,
             int32_t* cu_seqlens, int num_reqs, int64_t num_tokens, int max_blocks_per_seq, int block_size, bool capped, void* stream) {
    if (num_reqs < 0 || num_reqs > (1 << 30) || num_tokens < 0 || num_tokens > 0x7fffffffLL || max_blocks_per_seq <= 0 || num_free < 0 || num_free > 0x7fffffffLL ||
        block_table_stride < max_blocks_per_seq)
        return FQ_ERR_BAD_SHAPE;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (int64_t(max_blocks_per_seq) * block_size > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    if (!free_end || !cu_seqlens || (num_reqs > 0 && (!context_lens || !query_lens || !block_table || !seq_lens)) ||
        (num_free > 0 && !free_blocks) || (num_tokens > 0 && (!slot_mapping || !positions)))
        return FQ_ERR_NULL_POINTER;
    if (free_end == free_start) return FQ_ERR_BAD_SHAPE;      // one workgroup would write what others read
    fq::ScheduleParams p;
    p.context = context_lens; p.query = query_lens; p.table = block_table; p.free_blocks = free_blocks;
    p.free_start = free_start; p.free_end = free_end; p.slots = slot_mapping; p.positions = positions;
    p.seq_lens = seq_lens; p.cu = cu_seqlens; p.table_row = block_table_stride; p.num_tokens = num_tokens;
    p.S = num_reqs; p.max_blocks = max_blocks_per_seq; p.num_free = int(num_free);
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.capped = capped;
    const int64_t groups = (num_tokens + fq::kScheduleThreads - 1) / fq::kScheduleThreads;
    const unsigned grid = unsigned(groups > 0 ? groups : 1);
    hipStream_t s = static_cast<hipStream_t>(stream);
    // 256 requests: 3.1 us, 3.7 in the form for more; 1500, 36,000 tokens: 5.4 us, 6.9 in the form for few
    if (num_reqs <= fq::kScheduleThreads) fq::paged_schedule_kernel<1><<<grid, fq::kScheduleThreads, 0, s>>>(p);
    else fq::paged_schedule_kernel<fq::kScheduleMost><<<grid, fq::kScheduleThreads, 0, s>>>(p);
    return fq_host::check_launch();
}

}  // namespace

extern "C" int fq_paged_schedule(const int32_t* context_lens, const int32_t* query_lens, int32_t* block_table, int64_t block_table_stride,
                                 const int32_t* free_blocks, int64_t num_free, const int32_t* free_start, int32_t* free_end,
                                 int64_t* slot_mapping, int64_t* positions, int32_t* seq_lens, int32_t* cu_seqlens, int num_reqs,
                                 int64_t num_tokens, int max_blocks_per_seq, int block_size, void* stream) {
    return schedule(context_lens, query_lens, block_table, block_table_stride, free_blocks, num_free, free_start, free_end, slot_mapping, positions,
                    seq_lens, cu_seqlens, num_reqs, num_tokens, max_blocks_per_seq, block_size, false, stream);
}

extern "C" int fq_paged_schedule_capped(const int32_t* context_lens, const int32_t* query_lens, int32_t* block_table, int64_t block_table_stride,
                                        const int32_t* free_blocks, int64_t num_free, const int32_t* free_start, int32_t* free_end,
                                        int64_t* slot_mapping, int64_t* positions, int32_t* seq_lens, int32_t* cu_seqlens, int num_reqs,
                                        int64_t num_tokens, int max_blocks_per_seq, int block_size, void* stream) {
    return schedule(context_lens, query_lens, block_table, block_table_stride, free_blocks, num_free, free_start, free_end, slot_mapping, positions,
                    seq_lens, cu_seqlens, num_reqs, num_tokens, max_blocks_per_seq, block_size, true, stream);
}

extern "C" int fq_paged_advance(const int32_t* seq_lens, const int32_t* free_end, int num_blocks, int32_t* context_lens, int32_t* free_start,
                                const int32_t* cu_seqlens, const int64_t* positions, const int32_t* block_table, int64_t block_table_stride,
                                int32_t* token_table, int32_t* token_lens, int num_reqs, int64_t num_tokens, int max_blocks_per_seq,
                                int block_size, void* stream) {
    return fq_paged_advance_prefix(seq_lens, free_end, num_blocks, context_lens, free_start, cu_seqlens, positions, block_table, block_table_stride,
                                   nullptr, token_table, token_lens, nullptr, num_reqs, num_tokens, max_blocks_per_seq, block_size, stream);
}

extern "C" int fq_paged_advance_prefix(const int32_t* seq_lens, const int32_t* free_end, int num_blocks, int32_t* context_lens,
                                       int32_t* free_start, const int32_t* cu_seqlens, const int64_t* positions, const int32_t* block_table,
                                       int64_t block_table_stride, const int32_t* prefix_ids, int32_t* token_table, int32_t* token_lens,
                                       int32_t* token_prefix, int num_reqs, int64_t num_tokens, int max_blocks_per_seq, int block_size,
                                       void* stream) {
    if (num_reqs < 0 || num_reqs > (1 << 30) || num_blocks < 0 || num_tokens < 0 || num_tokens > 0x7fffffffLL || max_blocks_per_seq <= 0 ||
        block_table_stride < max_blocks_per_seq || (num_reqs == 0 && num_tokens > 0))
        return FQ_ERR_BAD_SHAPE;
    if (block_size != 8 && block_size != 16 && block_size != 32) return FQ_ERR_UNSUPPORTED_BLOCK;
    if (int64_t(max_blocks_per_seq) * block_size > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    if (!free_end || !free_start || (num_reqs > 0 && (!seq_lens || !context_lens)) ||
        (num_tokens > 0 && (!cu_seqlens || !positions || !block_table || !token_table || !token_lens || (token_prefix && !prefix_ids))))
        return FQ_ERR_NULL_POINTER;
    fq::AdvanceParams p;
    p.seq_lens = seq_lens; p.free_end = free_end; p.context = context_lens; p.free_start = free_start;
    p.cu = cu_seqlens; p.positions = positions; p.table = block_table; p.token_table = token_table; p.token_lens = token_lens;
    p.prefix_ids = prefix_ids; p.token_prefix = token_prefix;
    p.table_row = block_table_stride;
    p.S = num_reqs; p.max_blocks = max_blocks_per_seq; p.num_blocks = num_blocks;
    p.page_log2 = block_size == 8 ? 3 : block_size == 16 ? 4 : 5;
    p.state_groups = num_reqs > 0 ? (num_reqs + fq::kScheduleThreads - 1) / fq::kScheduleThreads : 1;
    p.parts = (max_blocks_per_seq + fq::kRowEntries - 1) / fq::kRowEntries;
    const int64_t groups = p.state_groups + num_tokens * p.parts;
    if (groups > 0x7fffffffLL) return FQ_ERR_BAD_SHAPE;
    fq::paged_advance_kernel<<<unsigned(groups), fq::kScheduleThreads, 0, static_cast<hipStream_t>(stream)>>>(p);
    return fq_host::check_launch();
}
