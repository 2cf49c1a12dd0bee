// svsx_attention.hip -- attention of one new token over paged rows (include/svsx.h: svsx_paged_attention_device).
#include "svsx_host.h"
#include "svsx_mfma.h"
#include <initializer_list>

namespace svsx {
namespace {

struct AttentionArgs {
    const void* queries;
    const void* keys;
    const void* values;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* sequences;
    void* out;
    float* lse;
    size_t query_stride, query_head_stride, key_page_stride, key_head_stride, key_row_stride, value_page_stride, value_head_stride, value_row_stride, table_stride;
    uint32_t n_queries, n_heads, group, n_key_heads, dk, dv, n_pages, page_size, n_sequences, max_pages;
    float scale;
    int shared;       // rows are keys and values at once
    int wide_queries, wide_out; // heads' queries, and heads' results, begin at 16-byte boundaries and are whole 16-byte words
};

// rows of query i: its table row and how many rows there are
__device__ __forceinline__ uint32_t rows_of(const AttentionArgs& a, uint32_t i, const int32_t** table) {
    const int32_t s = a.sequences ? a.sequences[i] : static_cast<int32_t>(i);
    if (s < 0 || static_cast<uint32_t>(s) >= a.n_sequences || a.n_pages == 0) return 0; // rows of a hole are read from page 0, and masked: there has to be one
    *table = a.table + static_cast<size_t>(s) * a.table_stride;
    const int32_t len = a.lengths[s];
    const uint32_t most = a.max_pages * a.page_size;
    return len <= 0 ? 0u : static_cast<uint32_t>(len) < most ? static_cast<uint32_t>(len) : most;
}

template <typename T> __global__ __launch_bounds__(256) void attend_head_kernel(const AttentionArgs a) {
    __shared__ RowsShared sm;
    const uint32_t h = blockIdx.x, i = blockIdx.y, g = h / a.group;
    const int32_t* table = nullptr;
    const uint32_t n = rows_of(a, i, &table);
    const T* q = static_cast<const T*>(a.queries) + i * a.query_stride + h * a.query_head_stride;
    for (uint32_t c = threadIdx.x; c < a.dk; c += 256) sm.q[c] = to_f32(q[c]);
    __syncthreads();
    const T* keys = static_cast<const T*>(a.keys) + g * a.key_head_stride;
    const T* values = static_cast<const T*>(a.values) + g * a.value_head_stride;
    auto page_of = [&](uint32_t r) { return table[r / a.page_size]; };
    auto key_of = [&](uint32_t r) -> const T* {
        const int32_t p = page_of(r);
        return p < 0 || static_cast<uint32_t>(p) >= a.n_pages ? nullptr : keys + p * a.key_page_stride + (r % a.page_size) * a.key_row_stride;
    };
    auto value_of = [&](uint32_t r) { return values + page_of(r) * a.value_page_stride + (r % a.page_size) * a.value_row_stride; };
    const float lse = attend_rows<T>(sm, n, a.dk, a.dv, a.scale, key_of, value_of);
    T* out = static_cast<T*>(a.out) + (static_cast<size_t>(i) * a.n_heads + h) * a.dv;
    for (uint32_t c = threadIdx.x; c < a.dv; c += 256) out[c] = from_f32<T>(sm.out[0][c]);
    if (a.lse && threadIdx.x == 0) a.lse[static_cast<size_t>(i) * a.n_heads + h] = lse;
}

// ---- heads that share a key head, on the matrix units --------------------------------------------------------------------------------------------
//
// One wave takes 32 rows of one key head at a time for up to 16 query heads that share it; what it needs of them goes from HBM to registers once and is not
// staged in LDS (variants whose registers do not hold it all spill: below):
//   S = K Q^T      rows x heads.  Row m of the s-th 16 x 16 product is row (m / 4) * 8 + s * 4 + m % 4 of the 32, so that lane l gets the scores of the EIGHT
//                  CONSECUTIVE rows 8 (l / 16) .. + 7 for head l % 16.
//   O^T = V^T P^T  columns x heads.  The lane's eight probabilities are a fragment of P^T as they are; and since it owns eight consecutive rows, it loads 8 columns
//                  (16 bytes) of each of them and transposes that 8 x 8 block in its registers: lane l's columns are 8 (l % 16) .. + 7, the d-th product
//                  takes the d-th of them.
// Bound by HBM: 16 heads' products are half the matrix units' time per byte, and 32 rows' keys (of the next 32) and values are in flight per wave, three waves per SIMD.
// 4 sequences of 131071 rows, 64 heads on 8 (2.15 GB, bfloat16): 384 us, 5.6 TB/s; 64 of up to 8191 rows, 32 heads on 8 (float16; 1.04 to 1.25 GB by the lengths drawn): 211 to 246 us, 5.0 TB/s; a
// kernel that only reads reached 6.3 TB/s.
// Registers: rows of up to 128 aligned 16-bit columns in pages of a multiple of 8 fit, but for 15 spilled at 128 columns.  32 sequences of 4096 rows, 32 heads on 8, spilled registers and rate: bfloat16 128
// columns 16, 4.6 TB/s; 192 28, 4.3; 256 71, 3.8; pages of 5 rows 100, 3.0; rows that are not aligned, 100 columns 48, 1.0; float32 128 columns 4, 5.5; 192 405, 2.9; 256 521, 2.9; 256 not aligned
// 1780, 0.9; pages of 5 rows 44, 4.0.
// The running maximum of a head is raised only when a score exceeds it by more than 2^kSlack (the accumulators are rescaled then), so the usual 32 rows cost
// no rescaling; sums are kept per lane and joined at the end.
//
// A workgroup is four waves that deal the tiles of one chunk of rows among themselves.  Chunks: see plan below.

constexpr int kTile = 32, kChunkUnit = 4 * kTile; // rows of a wave's tile; rows that a workgroup takes at a time

struct Plan {
    float* partial;  // [slot][head][dv] sums of p v
    float2* stats;   // [slot][head] {maximum (powers of two), sum of p}
    int2* chunks;    // [query] {first slot, chunks}
    uint32_t workers; // workgroups that share all rows; 0: one workgroup a query and no joining
    uint32_t unit;    // rows that a workgroup takes at a time
};

// Which rows a workgroup has.  Lengths are known on the device only, so every workgroup derives the same plan from them: all queries' rows, in units of plan.unit, one
// query behind the other, are cut into `workers` equal runs; a workgroup takes its run query by query.  Worker w's part of query i goes to slot w + i: along the line of
// units each step raises one of the two, so slots differ, and a query's are consecutive (at most workers + n_queries slots).
struct Chunk {
    uint32_t query, begin, end, slot, count; // count: parts of this query; 1: nothing to join
    const int32_t* table;
};
template <uint32_t kThreads> struct Walk {
    static constexpr uint32_t kWaves = kThreads / 64;
    uint32_t total, workers, stop, query, before; // all units; workers that have some; the end of this worker's run; units before the query's first

    static __device__ __forceinline__ uint32_t units(const AttentionArgs& a, const Plan& plan, uint32_t i) {
        const int32_t* unused;
        return i < a.n_queries ? (rows_of(a, i, &unused) + plan.unit - 1) / plan.unit : 0u;
    }
    // the worker whose run [floor(w total / workers), floor((w + 1) total / workers)) has unit u
    __device__ __forceinline__ uint32_t owner(uint32_t u) const { return static_cast<uint32_t>(((u + 1ull) * workers - 1) / total); }

    __device__ __forceinline__ void set(const AttentionArgs& a, const Plan& plan, uint32_t unit, Chunk* c) {
        c->query = query;
        c->table = nullptr;
        const uint32_t rows = __builtin_amdgcn_readfirstlane(rows_of(a, query, &c->table)), mine = (rows + plan.unit - 1) / plan.unit;
        const uint32_t first = owner(before);
        c->begin = __builtin_amdgcn_readfirstlane((unit - before) * plan.unit);
        c->end = __builtin_amdgcn_readfirstlane(min(rows, (min(before + mine, stop) - before) * plan.unit));
        c->slot = blockIdx.x + query;
        c->count = __builtin_amdgcn_readfirstlane(owner(before + mine - 1) - first + 1);
        if (unit == before && threadIdx.x == 0 && blockIdx.y == 0) plan.chunks[query] = make_int2(static_cast<int>(first + query), static_cast<int>(c->count));
    }
    // the first part of this worker's run; false: it has none
    __device__ __forceinline__ bool first(const AttentionArgs& a, const Plan& plan, Chunk* c, uint32_t (&sh)[24]) {
        if (plan.workers == 0) {
            c->query = blockIdx.x;
            c->table = nullptr;
            c->begin = 0;
            c->end = __builtin_amdgcn_readfirstlane(rows_of(a, c->query, &c->table));
            c->slot = 0;
            c->count = 1;
            return true;
        }
        const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63;
        auto scan = [&](uint32_t n, uint32_t base, uint32_t* all) { // units before this thread's query, after `base` of them; two barriers
            uint32_t incl = n;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t u = __shfl_up(incl, off);
                if (lane >= static_cast<uint32_t>(off)) incl += u;
            }
            __syncthreads();
            if (lane == 63) sh[wave] = incl;
            __syncthreads();
            uint32_t at = base + incl - n;
            *all = base;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                const uint32_t some = __builtin_amdgcn_readfirstlane(sh[w]);
                at += w < wave ? some : 0;
                *all += some;
            }
            return at;
        };
        // all that follows waits for one load, for up to kThreads queries
        const uint32_t mine = units(a, plan, t);
        uint32_t n = mine, at = scan(mine, 0, &total), upto = total;
        for (uint32_t from = kThreads; from < a.n_queries; from += kThreads) scan(units(a, plan, from + t), total, &total);
        workers = min(plan.workers, total); // no run is empty: a query's parts are those of consecutive workers
        if (blockIdx.x >= workers) return false;
        const uint32_t start = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(blockIdx.x) * total / workers));
        stop = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>((blockIdx.x + 1ull) * total / workers));
        for (uint32_t from = 0;;) { // which query has the first unit
            if (n > 0 && start >= at && start < at + n) {
                sh[16] = from + t;
                sh[17] = at;
            }
            from += kThreads;
            if (upto > start || from >= a.n_queries) break;
            n = units(a, plan, from + t);
            at = scan(n, upto, &upto);
        }
        __syncthreads();
        query = __builtin_amdgcn_readfirstlane(sh[16]); // the same for all: in scalar registers, so that loops over it are too
        before = __builtin_amdgcn_readfirstlane(sh[17]);
        set(a, plan, start, c);
        return true;
    }
    // the next one
    __device__ __forceinline__ bool next(const AttentionArgs& a, const Plan& plan, Chunk* c) {
        if (plan.workers == 0) return false;
        uint32_t mine = __builtin_amdgcn_readfirstlane(units(a, plan, query));
        if (before + mine >= stop) return false;
        do { // units are left, so there is a query that has them
            before += mine;
            ++query;
            mine = __builtin_amdgcn_readfirstlane(units(a, plan, query));
        } while (mine == 0 && query < a.n_queries);
        set(a, plan, before, c);
        return true;
    }
};

// The lane, as something that the compiler cannot know to be the same for every part of a worker's run: what follows from it would otherwise be kept in registers over
// the whole run (addresses and conditions of code that runs once a part), and there are none to spare.
__device__ __forceinline__ uint32_t lane_here() {
    uint32_t lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Where a lane's rows are: pages of the two key rows and the eight value rows.  Page8: page_size is a multiple of 8, so eight consecutive rows share a page.
template <bool Page8> struct TileRows {
    int32_t key[Page8 ? 1 : 2], value[Page8 ? 1 : 8];
    uint32_t key_at[Page8 ? 1 : 2], value_at[Page8 ? 1 : 8]; // row within the page
};

template <typename T, int KS, int VB, bool Wide, bool Page8>
__global__ __launch_bounds__(256, sizeof(T) == 2 && VB == 1 ? 3 : 2) void attend_group_kernel(const AttentionArgs a, const Plan plan, const Divider by_page) {
    __shared__ uint32_t sh[24];
    __shared__ float join[2][VB * 32 + 2][64];
    Chunk c;
    Walk<256> walk;
    if (!walk.first(a, plan, &c, sh)) return;
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t tiles = (a.group + 15) / 16, g = blockIdx.y / tiles, h0 = (blockIdx.y % tiles) * 16; // key head; first head within its group
    const uint32_t heads = min(16u, a.group - h0);

    do {
        const uint32_t lane = lane_here(), n = lane & 15, quad = lane >> 4, head = g * a.group + h0 + n;
        const bool live = n < heads;
        Frag<T> q[KS];
        {
            const T* row = static_cast<const T*>(a.queries) + c.query * a.query_stride + (live ? head : g * a.group) * a.query_head_stride;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                q[k] = a.wide_queries ? load_frag<T, true>(row, k * 32 + quad * 8, a.dk) : load_frag<T, false>(row, k * 32 + quad * 8, a.dk);
                if (!live) q[k] = Frag<T>{};
            }
        }
        const T* keys = static_cast<const T*>(a.keys) + g * a.key_head_stride;
        const T* values = static_cast<const T*>(a.values) + g * a.value_head_stride;
        const float scale = a.scale * kLog2e;

        f32x4 o[VB * 8];
#pragma unroll
        for (int i = 0; i < VB * 8; ++i) o[i] = f32x4{0, 0, 0, 0};
        float top = -INFINITY, sum = 0.0f; // the maximum that probabilities are relative to, in powers of two; this lane's share of their sum

        const uint32_t last = c.end - 1; // rows behind the end are looked up at the last one, and masked
        auto find = [&](uint32_t base) {
            TileRows<Page8> r;
            if constexpr (Page8) {
                r.key[0] = c.table[by_page(min(base + (n >> 2) * 8, last), &r.key_at[0])];
                r.value[0] = c.table[by_page(min(base + quad * 8, last), &r.value_at[0])];
                // the page's row of the block's first row: `last` may be in its middle
                r.key_at[0] &= ~7u;
                r.value_at[0] &= ~7u;
            } else {
#pragma unroll
                for (int s = 0; s < 2; ++s) r.key[s] = c.table[by_page(min(base + (n >> 2) * 8 + s * 4 + (n & 3), last), &r.key_at[s])];
#pragma unroll
                for (int j = 0; j < 8; ++j) r.value[j] = c.table[by_page(min(base + quad * 8 + j, last), &r.value_at[j])];
            }
            return r;
        };
        auto is_page = [&](int32_t p) { return static_cast<uint32_t>(p) < a.n_pages; }; // negative ones are large
        auto load_keys = [&](const TileRows<Page8>& r, Frag<T> (&k)[2][KS]) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int32_t p = Page8 ? r.key[0] : r.key[Page8 ? 0 : s];
                const uint32_t at = Page8 ? r.key_at[0] + s * 4 + (n & 3) : r.key_at[Page8 ? 0 : s];
                const T* row = keys + (is_page(p) ? static_cast<size_t>(p) : 0) * a.key_page_stride + at * a.key_row_stride;
#pragma unroll
                for (int i = 0; i < KS; ++i) k[s][i] = load_frag<T, Wide>(row, i * 32 + quad * 8, a.dk);
            }
        };

        uint32_t base = c.begin + wave * kTile;
        Frag<T> k[2][KS];
        TileRows<Page8> here, next;
        if (base < c.end) {
            here = find(base);
            load_keys(here, k);
            next = find(base + kChunkUnit);
        }
        for (; base < c.end; base += kChunkUnit) {
            Frag<T> v[VB][8];
            uint32_t mask = 0; // which of the lane's eight rows are there
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int32_t p = Page8 ? here.value[0] : here.value[Page8 ? 0 : j];
                const uint32_t at = Page8 ? here.value_at[0] + j : here.value_at[Page8 ? 0 : j];
                if (base + quad * 8 + j < c.end && is_page(p)) mask |= 1u << j;
                const T* row = values + (is_page(p) ? static_cast<size_t>(p) : 0) * a.value_page_stride + at * a.value_row_stride;
#pragma unroll
                for (int b = 0; b < VB; ++b) v[b][j] = load_frag<T, Wide>(row, b * 128 + n * 8, a.dv);
            }
            f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                s[0] = product16(k[0][i], q[i], s[0]);
                s[1] = product16(k[1][i], q[i], s[1]);
            }
            if (base + kChunkUnit < c.end) {
                here = next;
                load_keys(here, k);
                next = find(base + 2 * kChunkUnit);
            }
            float p[8], most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = s[j >> 2][j & 3] * scale;
            if (!__all(mask == 0xFFu)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool there = mask >> j & 1;
                    p[j] = there ? p[j] : -INFINITY;
#pragma unroll
                    for (int b = 0; b < VB; ++b) // what a page holds behind the last row is not defined: zero times it need not be zero
                        if (!there) v[b][j] = Frag<T>{};
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, p[j]);
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            if (__any(most > top + kSlack)) { // also the first tile: top is -inf
                const float raised = fmaxf(top, most), shrink = top == -INFINITY ? 0.0f : exp2_fast(top - raised);
                top = raised;
                sum *= shrink;
#pragma unroll
                for (int i = 0; i < VB * 8; ++i) o[i] *= shrink;
            }
            const float from = (top == -INFINITY ? 0.0f : top) - kLift<T>;
            Frag<T> w;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = exp2_fast(p[j] - from);
                sum += p[j];
                w[j] = from_f32<T>(p[j]);
            }
#pragma unroll
            for (int b = 0; b < VB; ++b) {
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    Frag<T> column;
#pragma unroll
                    for (int j = 0; j < 8; ++j) column[j] = v[b][j][d];
                    o[b * 8 + d] = product16(column, w, o[b * 8 + d]);
                }
            }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        top -= kLift<T>; // sums are of 2^(score - top)

        // the four waves' results, two at a time: waves 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
        for (int half = 2; half >= 1; half >>= 1) {
            __syncthreads();
            if (wave >= static_cast<uint32_t>(half) && wave < 2u * half) {
#pragma unroll
                for (int i = 0; i < VB * 32; ++i) join[wave - half][i][lane] = o[i >> 2][i & 3];
                join[wave - half][VB * 32][lane] = top;
                join[wave - half][VB * 32 + 1][lane] = sum;
            }
            __syncthreads();
            if (wave < static_cast<uint32_t>(half)) {
                const float other = join[wave][VB * 32][lane], all = fmaxf(top, other);
                const float wa = top == -INFINITY ? 0.0f : exp2_fast(top - all), wb = other == -INFINITY ? 0.0f : exp2_fast(other - all);
                sum = sum * wa + join[wave][VB * 32 + 1][lane] * wb;
                top = all;
#pragma unroll
                for (int i = 0; i < VB * 32; ++i) o[i >> 2][i & 3] = o[i >> 2][i & 3] * wa + join[wave][i][lane] * wb;
            }
        }
        if (wave != 0 || !live) continue;
        // o[b * 8 + d][r]: column b * 128 + (quad * 4 + r) * 8 + d of head n
        if (c.count > 1) {
            const size_t at = static_cast<size_t>(c.slot) * a.n_heads + head;
            if (quad == 0) plan.stats[at] = make_float2(top, sum);
            float* out = plan.partial + at * a.dv;
#pragma unroll
            for (int b = 0; b < VB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        const uint32_t col = b * 128 + (quad * 4 + r) * 8 + d;
                        if (col < a.dv) out[col] = o[b * 8 + d][r];
                    }
            continue;
        }
        const size_t at = static_cast<size_t>(c.query) * a.n_heads + head;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* out = static_cast<T*>(a.out) + at * a.dv;
#pragma unroll
        for (int b = 0; b < VB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t col = b * 128 + (quad * 4 + r) * 8;
                Frag<T> f;
#pragma unroll
                for (int d = 0; d < 8; ++d) f[d] = from_f32<T>(o[b * 8 + d][r] * inv);
                if (a.wide_out) {
                    if (col < a.dv) *reinterpret_cast<Frag<T>*>(out + col) = f;
                } else {
#pragma unroll
                    for (uint32_t d = 0; d < 8; ++d)
                        if (col + d < a.dv) out[col + d] = f[d];
                }
            }
        if (a.lse && quad == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    } while (walk.next(a, plan, &c));
}

// ---- few rows, a head a key head ------------------------------------------------------------------------------------------------------------------
//
// Attention over the answers of a search: at most a few hundred rows, each somewhere else, for one head.  There is nothing to split and nothing for the matrix
// units to share; what counts is how many rows are on their way at once.  One wave takes a query (of one key head): 16 lanes a row, 8 or 16 columns a lane, so four rows
// at a time; 64 table entries are looked up by the 64 lanes at once; each 16 lanes keep a softmax of their own, joined at the end.
// 2048 queries of 100 rows of 96 float32 columns, keys and values apart (157 MB read): 22 us from a set of 15 MB, which the caches hold (48 us through attend_group_kernel, whose four waves a query have one
// tile each); 27 us from a million rows, 45 G lines/s of 128 bytes of the 49 that random reads reach.  Rows that are key and value at once, a million: 18 us, 34 G lines/s; bfloat16 16 us.
// float16, 128 columns, few against group: 512 queries of 64 rows 8.9 and 12.0 us, of 256 rows 24 and 34, of 512 rows 44 and 55, of 1024 rows 84.5 and 83.5; 128 queries of 64 rows 9.0 and 9.0, of
// 256 rows 21.5 and 17.3.  With two heads a key head and 8 key heads it is the slower one from 4096 waves on.

constexpr uint32_t kFewRows = 512, kFewItems = 512; // at most so many rows a query; at least so many waves

// sum over the 16 lanes of a row of the wave, for each of them
__device__ __forceinline__ float sum16(float x) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF, false)); // rotated by 8, 4, 2, 1
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xF, 0xF, false));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xF, 0xF, false));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xF, 0xF, false));
    return x;
}

template <typename T, int E, bool Wide> __global__ __launch_bounds__(256) void attend_few_kernel(const AttentionArgs a, const Divider by_page) {
    constexpr int kBatch = E == 8 ? 8 : 4, kFrags = E / 8; // rows that each 16 lanes have on their way
    const uint32_t lane = threadIdx.x & 63, item = blockIdx.x * 4 + (threadIdx.x >> 6), quarter = lane >> 4, n16 = lane & 15;
    if (item >= a.n_queries * a.n_key_heads) return;
    const uint32_t i = item / a.n_key_heads, g = item % a.n_key_heads;
    const int32_t* table = nullptr;
    const uint32_t n = __builtin_amdgcn_readfirstlane(rows_of(a, i, &table));
    const T* keys = static_cast<const T*>(a.keys) + g * a.key_head_stride;
    const T* values = static_cast<const T*>(a.values) + g * a.value_head_stride;
    const float scale = a.scale * kLog2e;
    float q[E], o[E], top = -INFINITY, sum = 0.0f;
    const T* const query = static_cast<const T*>(a.queries) + i * a.query_stride + g * a.query_head_stride;
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
        const Frag<T> x = a.wide_queries ? load_frag<T, true>(query, n16 * E + f * 8, a.dk) : load_frag<T, false>(query, n16 * E + f * 8, a.dk);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q[f * 8 + e] = to_f32(x[e]);
            o[f * 8 + e] = 0.0f;
        }
    }
    for (uint32_t base = 0; base < n; base += 64) {
        uint32_t at;
        const int32_t mine = table[by_page(min(base + lane, n - 1), &at)];
        const bool is = base + lane < n && static_cast<uint32_t>(mine) < a.n_pages;
        const int32_t page = is ? mine : -1;
        for (uint32_t first = 0; first < 16 && base + first * 4 < n; first += kBatch) {
            Frag<T> k[kBatch][kFrags], v[kBatch][kFrags];
            bool there[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int from = static_cast<int>((first + j) * 4 + quarter);
                const int32_t p = __shfl(page, from);
                const uint32_t r = __shfl(at, from);
                there[j] = p >= 0;
                const T* row = keys + (p >= 0 ? static_cast<size_t>(p) : 0) * a.key_page_stride + r * a.key_row_stride;
#pragma unroll
                for (int f = 0; f < kFrags; ++f) k[j][f] = load_frag<T, Wide>(row, n16 * E + f * 8, a.dk);
                if (!a.shared) {
                    const T* vrow = values + (p >= 0 ? static_cast<size_t>(p) : 0) * a.value_page_stride + r * a.value_row_stride;
#pragma unroll
                    for (int f = 0; f < kFrags; ++f) v[j][f] = load_frag<T, Wide>(vrow, n16 * E + f * 8, a.dv);
                }
            }
            float s[kBatch], most = top;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) x = fmaf(to_f32(k[j][e >> 3][e & 7]), q[e], x);
                s[j] = there[j] ? sum16(x) * scale : -INFINITY;
                most = fmaxf(most, s[j]);
            }
            const float ref = most == -INFINITY ? 0.0f : most, was = exp2_fast(top - ref);
            top = most;
            sum *= was;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= was;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const float p = exp2_fast(s[j] - ref);
                sum += p;
                if (there[j]) { // what a row that is not there would be read from is not defined
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(p, to_f32(a.shared ? k[j][e >> 3][e & 7] : v[j][e >> 3][e & 7]), o[e]);
                }
            }
        }
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
        const float other = __shfl_xor(top, off), all = fmaxf(top, other);
        const float mine = top == -INFINITY ? 0.0f : exp2_fast(top - all), theirs = other == -INFINITY ? 0.0f : exp2_fast(other - all);
        sum = sum * mine + __shfl_xor(sum, off) * theirs;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * mine + __shfl_xor(o[e], off) * theirs;
        top = all;
    }
    if (quarter != 0) return;
    const size_t at = static_cast<size_t>(i) * a.n_heads + g;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out) + at * a.dv;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e)
        if (n16 * E + e < a.dv) out[n16 * E + e] = from_f32<T>(o[e] * inv);
    if (a.lse && n16 == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// ---- rows that are key and value at once, for many heads ------------------------------------------------------------------------------------------
//
// Latent rows: every head reads the same row, as key and (its first columns) as value, so 64 heads make 240 operations of each byte and the rows have to be
// read from HBM once for all of them.  A workgroup brings 64 rows into LDS (straight from HBM, two buffers: the next 64 arrive while these are worked on) and
// takes up to 64 heads over them, with eight waves (four for 16 heads):
//   S = K Q^T     a wave takes 16 or 32 of the rows for 16 of the heads; its queries stay in registers
//   maximum of the 64 rows per head through LDS; P, rounded to the row type, through LDS
//   O^T = V^T P^T a wave takes its share of the value columns for all rows and heads; the transposed fragments come from gfx950's transposing LDS reads
// (float32 rows: single words).  No sums are joined between waves but that of the probabilities.
// LDS holds a row as 16-byte words in planes of 64 words, rows 32 bytes further apart than they are long, so that neither eight rows of a key fragment nor the 16
// half-words of a transposed one meet in a bank; and a narrow plane for the rest, which is brought in several rows at a time and has its words exchanged in fours instead.
// (Exchanging single words of the long rows as well, with no padding, was measured: the loads then cross each 64-byte line out of order and cost twice the time.)
// 32 sequences of up to 8192 rows, 128 heads (about 37 GFLOP, 160 to 175 MB by the lengths drawn, bfloat16): 90 to 101 us, 390 TFLOP/s; one of 4097 rows, 16 heads: 17.7 us.
// float32 has one buffer and 16 heads a workgroup, so 128 heads bring the rows in eight times: 32 sequences of 4096 rows 579 us (104 with 16 heads); bfloat16 80 (36).
// At 16 heads HBM bounds it; at 64 the latency of the steps between a tile's barriers (LDS is busy for 2400 cycles of a tile's 8000, the matrix units for 2176, and the loads straight to LDS,
// which come to 30 bytes a cycle, for 2400).  Measured in place of it, 32 sequences, 128 heads: two workgroups of 32-row buffers and four waves on a compute unit, whose registers spill, 104 -> 127 us; four
// waves of 512 registers that take 32 rows for 32 heads and read LDS half as often, 98 -> 112 us, since a wave stands still while it gives out loads and no other wave is there.

template <typename T, int KS, int HT> struct RowsLayout { // KS: 32-column steps of a key row; HT: 16-head tiles
    static constexpr uint32_t kRows = 64;                                      // rows of a tile
    static constexpr int kWaves = HT == 1 ? 4 : 8, kThreads = kWaves * 64;
    static constexpr int DT = (KS > 10 ? 32 : 16) / kWaves;                    // 16-column value tiles of a wave: 512 or 256 columns in all
    static constexpr uint32_t kBring = kRows / kWaves;                         // rows that a wave brings in
    static constexpr int kWords = KS * 32 * sizeof(T) / 16;                    // 16-byte words in a row
    static constexpr int kPlanes = kWords < 64 ? 1 : kWords / 64, kTail = kWords < 64 ? 0 : kWords % 64;
    static constexpr uint32_t kPlaneRow = 1024 + 32, kPlaneBytes = kRows * kPlaneRow;
    static constexpr int kTileBytes = kPlaneBytes * kPlanes + kRows * 16 * kTail;
    static constexpr int kBuffers = sizeof(T) == 2 ? 2 : 1;                    // float32 rows: one buffer is 144 KB
    static constexpr uint32_t kProbRow = kRows * sizeof(T), kProbWords = kProbRow / 16;
    static constexpr int kProbBytes = HT * 16 * kProbRow;
    static constexpr int kTilesPerWave = HT == 4 ? 2 : 1;                      // of 16 rows, for one tile of 16 heads
    static constexpr int kParts = kRows / 16 / kTilesPerWave;                  // waves that share a head's rows
    static constexpr int kStatBytes = kParts * HT * 16 * 4;
    static constexpr int kBytes = kBuffers * kTileBytes + kProbBytes + kStatBytes + 64;
    static_assert(kWaves == HT * kParts, "a wave is a tile of heads and a part of the rows");
    static __device__ __forceinline__ uint32_t prob(uint32_t h, uint32_t word) { return h * kProbRow + (word ^ (h / (16 / kProbWords) & (kProbWords - 1))) * 16; }
    static_assert(kTail == 0 || kTail == 8 || kTail == 16, "a narrow plane of 8 or 16 words");
    static_assert(kBytes + 128 <= 160 * 1024, "LDS");
    // byte of word j of row r
    static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t j) {
        if (kTail > 0 && j >= kPlanes * 64) return kPlaneBytes * kPlanes + r * (kTail * 16) + ((j - kPlanes * 64) ^ narrow(r)) * 16;
        return (j >> 6) * kPlaneBytes + r * kPlaneRow + (j & 63) * 16;
    }
    static __device__ __forceinline__ uint32_t narrow(uint32_t r) { return kTail == 8 ? (r >> 1 & 1) << 2 : (r & 3) << 2; }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T, int KS, int HT> __global__ __launch_bounds__((RowsLayout<T, KS, HT>::kThreads)) void attend_rows_kernel(const AttentionArgs a, const Plan plan, const Divider by_page) {
    typedef RowsLayout<T, KS, HT> L;
    constexpr int DT = L::DT;
    constexpr uint32_t kThreads = L::kThreads, kBring = L::kBring;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ uint32_t sh[24];
    Chunk c;
    Walk<L::kThreads> walk;
    if (!walk.first(a, plan, &c, sh)) return;
    constexpr int kElems = 16 / sizeof(T); // elements in a 16-byte word
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t groups = (a.group + HT * 16 - 1) / (HT * 16), g = blockIdx.y / groups, h0 = (blockIdx.y % groups) * (HT * 16);
    const uint32_t heads = min(static_cast<uint32_t>(HT * 16), a.group - h0);
    unsigned char* probs = lds + L::kBuffers * L::kTileBytes;
    float* parts = reinterpret_cast<float*>(probs + L::kProbBytes); // [part][head]: maxima; sums
    uint32_t* masks = reinterpret_cast<uint32_t*>(probs + L::kProbBytes + L::kStatBytes); // [buffer][wave]: which of the rows that the wave brought in are there
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_byte*)lds));

    const uint32_t words = a.dk / kElems; // of a row in memory; what LDS holds beyond them has to be finite

    // the wave's queries: heads of tile ht, rows of tiles rt0 ..; through LDS, zeros where there is no head or column
    const uint32_t ht = wave % HT, rt0 = wave / HT * L::kTilesPerWave, part = wave / HT;
    static_assert(HT * 16 * KS * 32 * sizeof(T) <= L::kBuffers * L::kTileBytes, "LDS");
    do {
        const uint32_t lane = lane_here(), thread = wave * 64 + lane, n = lane & 15, quad = lane >> 4;
        Frag<T> q[KS];
        {
            const T* from = static_cast<const T*>(a.queries) + c.query * a.query_stride + (g * a.group + h0) * a.query_head_stride;
            T* stage = reinterpret_cast<T*>(lds);
            constexpr uint32_t kRow = KS * 32, kBatch = 9;
            if (a.wide_queries) {
                constexpr uint32_t kAll = HT * 16 * kRow / 8;
                for (uint32_t first = 0; first < kAll; first += kThreads * kBatch) {
                    Frag<T> f[kBatch];
#pragma unroll
                    for (uint32_t i = 0; i < kBatch; ++i) {
                        const uint32_t at = first + i * kThreads + thread, h = at / (kRow / 8), col = at % (kRow / 8) * 8;
                        f[i] = Frag<T>{};
                        if (h < heads && col < a.dk) f[i] = *reinterpret_cast<const Frag<T>*>(from + h * a.query_head_stride + col);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < kBatch; ++i)
                        if (const uint32_t at = first + i * kThreads + thread; at < kAll) *reinterpret_cast<Frag<T>*>(stage + at * 8) = f[i];
                }
            } else {
                for (uint32_t i = thread; i < HT * 16 * kRow; i += kThreads) {
                    const uint32_t h = i / kRow, col = i % kRow;
                    stage[i] = h < heads && col < a.dk ? from[h * a.query_head_stride + col] : from_f32<T>(0.0f);
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const Frag<T>*>(stage + (ht * 16 + n) * kRow + k * 32 + quad * 8);
            __syncthreads();
        }
        if (words < static_cast<uint32_t>(L::kWords)) {
            for (uint32_t i = thread; i < L::kBuffers * L::kTileBytes / 16; i += kThreads) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        f32x4 o[HT][DT];
#pragma unroll
        for (int x = 0; x < HT; ++x)
#pragma unroll
            for (int d = 0; d < DT; ++d) o[x][d] = f32x4{0, 0, 0, 0};
        float top[HT], sum = 0.0f;
#pragma unroll
        for (float& x : top) x = -INFINITY;
        const float scale = a.scale * kLog2e;
        const T* keys = static_cast<const T*>(a.keys) + g * a.key_head_stride;

        // rows that this wave brings in: kBring wave + n of a tile.  A row's page is looked up a tile before it is brought in, ahead of the loads that
        // are to stay in flight: loads come back in order, and what waits for the page would wait for them.
        const T* row = keys;
        uint32_t there = 0, page_row = 0;
        int32_t page = -1;
        auto look = [&](uint32_t base) { page = c.table[by_page(min(base + wave * kBring + n % kBring, c.end - 1), &page_row)]; };
        auto find = [&](uint32_t base) {
            const bool is = static_cast<uint32_t>(page) < a.n_pages;
            row = keys + (is ? static_cast<size_t>(page) : 0) * a.key_page_stride + page_row * a.key_row_stride;
            there = static_cast<uint32_t>(__ballot(is && base + wave * kBring + n % kBring < c.end)) & ((1u << kBring) - 1);
        };
        auto bring = [&](uint32_t buffer) {
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + buffer * L::kTileBytes);
            const uint64_t addr = reinterpret_cast<uint64_t>(row);
#pragma unroll
            for (uint32_t r = 0; r < kBring; ++r) {
                const uint64_t base = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(addr >> 32), r)) << 32 |
                                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(addr), r));
#pragma unroll
                for (uint32_t plane = 0; plane < static_cast<uint32_t>(L::kPlanes); ++plane) {
                    const uint32_t word = plane * 64 + lane;
                    if (words >= (plane + 1) * 64 || word < words) direct_load(reinterpret_cast<const void*>(base), word * 16, to + plane * L::kPlaneBytes + (wave * kBring + r) * L::kPlaneRow);
                }
            }
            if constexpr (L::kTail > 0) {
                constexpr uint32_t kRows = 64 / L::kTail; // rows in one go
#pragma unroll
                for (uint32_t r = 0; r < kBring; r += kRows) {
                    const uint32_t mine = r + lane / L::kTail;
                    const uint64_t base = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(addr >> 32), mine)) << 32 | __shfl(static_cast<uint32_t>(addr), mine);
                    const uint32_t word = L::kPlanes * 64 + (lane % L::kTail ^ L::narrow(mine));
                    const void* from = reinterpret_cast<const unsigned char*>(base) + word * 16;
                    const uint32_t dst = to + L::kPlaneBytes * L::kPlanes + (wave * kBring + r) * (L::kTail * 16);
                    if (word < words) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(from) : "memory", "m0");
                }
            }
        };
        // once the rows are there: rows that are not to be seen become zeros (a weight of zero times what a page holds behind the last row need not be zero)
        auto settle = [&](uint32_t buffer, uint32_t mask) {
            direct_wait();
            if (mask != (1u << kBring) - 1) {
                unsigned char* tile = lds + buffer * L::kTileBytes;
                for (uint32_t r = 0; r < kBring; ++r)
                    if (!(mask >> r & 1))
                        for (uint32_t j = lane; j < static_cast<uint32_t>(L::kWords); j += 64) *reinterpret_cast<uint4*>(tile + L::at(wave * kBring + r, j)) = make_uint4(0, 0, 0, 0);
            }
            if (lane == 0) masks[buffer * L::kWaves + wave] = mask;
        };

        uint32_t now = 0, mask = 0;
        if (c.begin < c.end) {
            look(c.begin);
            find(c.begin);
            look(c.begin + L::kRows);
            bring(0);
            mask = there;
            settle(0, mask);
            lds_barrier();
        }
        for (uint32_t base = c.begin; base < c.end; base += L::kRows) {
            const bool more = base + L::kRows < c.end;
            auto next = [&] {
                find(base + L::kRows);
                look(base + 2 * L::kRows);
                bring(now ^ 1);
                mask = there;
            };
            // giving out the loads takes a wave 1300 cycles: of the two waves of a SIMD one gives them out before its products of keys and the other after (104 -> 98 us, 32 sequences, 128 heads)
            if (L::kBuffers == 2 && more && !(wave & 4)) next();
            const unsigned char* tile = lds + now * L::kTileBytes;
            f32x4 s[L::kTilesPerWave];
#pragma unroll
            for (int t = 0; t < L::kTilesPerWave; ++t) s[t] = f32x4{0, 0, 0, 0};
            uint32_t key_at[L::kTilesPerWave], tail_at[L::kTilesPerWave]; // this lane's first word of its rows
            constexpr int kStep = 2 * sizeof(T);                          // words in 32 columns
#pragma unroll
            for (int t = 0; t < L::kTilesPerWave; ++t) {
                key_at[t] = L::at((rt0 + t) * 16 + n, quad * (kStep / 4));
                tail_at[t] = L::kTail ? L::at((rt0 + t) * 16 + n, L::kPlanes * 64 + quad * (kStep / 4)) : 0;
            }
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int t = 0; t < L::kTilesPerWave; ++t) {
                    const bool tail = k * kStep >= L::kPlanes * 64;
                    auto word = [&](uint32_t j) { return tile + (tail ? tail_at[t] ^ (j - L::kPlanes * 64) << 4 : key_at[t] + (j >> 6) * L::kPlaneBytes + (j & 63) * 16); };
                    Frag<T> f;
                    if constexpr (sizeof(T) == 2) {
                        f = *reinterpret_cast<const Frag<T>*>(word(k * kStep));
                    } else {
                        *reinterpret_cast<f32x4*>(&f) = *reinterpret_cast<const f32x4*>(word(k * kStep));
                        *(reinterpret_cast<f32x4*>(&f) + 1) = *reinterpret_cast<const f32x4*>(word(k * kStep + 1));
                    }
                    s[t] = product16(f, q[k], s[t]);
                }
            if (L::kBuffers == 2 && more && (wave & 4)) next();
            // lane: head n of tile ht, rows (rt0 + t) * 16 + quad * 4 + r
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < L::kTilesPerWave; ++t) {
                const uint32_t first = (rt0 + t) * 16 + quad * 4, seen = masks[now * L::kWaves + first / kBring] >> (first % kBring);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[t][r] = seen >> r & 1 ? s[t][r] * scale : -INFINITY;
                    most = fmaxf(most, s[t][r]);
                }
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const uint32_t h = ht * 16 + n;
            if (quad == 0) parts[part * (HT * 16) + h] = most;
            lds_barrier();
#pragma unroll
            for (int x = 0; x < HT; ++x) { // every wave keeps every head's maximum, from the same numbers
                most = parts[x * 16 + n];
#pragma unroll
                for (int i = 1; i < L::kParts; ++i) most = fmaxf(most, parts[i * (HT * 16) + x * 16 + n]);
                if (__any(most > top[x] + kSlack)) {
                    const float raised = fmaxf(top[x], most), shrink = top[x] == -INFINITY ? 0.0f : exp2_fast(top[x] - raised);
                    top[x] = raised;
                    if (ht == static_cast<uint32_t>(x)) sum *= shrink;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[x][d] *= shrink;
                }
            }
            float ref = top[0];
#pragma unroll
            for (int x = 1; x < HT; ++x) ref = ht == static_cast<uint32_t>(x) ? top[x] : ref;
            const float from = (ref == -INFINITY ? 0.0f : ref) - kLift<T>;
#pragma unroll
            for (int t = 0; t < L::kTilesPerWave; ++t) {
                typedef T Four __attribute__((ext_vector_type(4)));
                Four w;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = exp2_fast(s[t][r] - from);
                    sum += p;
                    w[r] = from_f32<T>(p);
                }
                const uint32_t at = ((rt0 + t) * 16 + quad * 4) * sizeof(T); // byte of the first of the four rows
                *reinterpret_cast<Four*>(probs + L::prob(h, at >> 4) + (at & 15)) = w;
            }
            lds_barrier();
            uint32_t value_at[2]; // row of the first 32, the wave's first columns
#pragma unroll
            for (int half = 0; half < 2; ++half) value_at[half] = L::at(quad * 8 + half * 4 + (n >> 2), wave * (DT * 2) + (n >> 1 & 1)) + (n & 1) * 8;
#pragma unroll
            for (int b = 0; b < L::kRows / 32; ++b) {
                Frag<T> w[HT];
#pragma unroll
                for (int x = 0; x < HT; ++x) {
                    const uint32_t h = x * 16 + n;
                    if constexpr (sizeof(T) == 2) {
                        w[x] = *reinterpret_cast<const Frag<T>*>(probs + L::prob(h, b * 4 + quad));
                    } else {
                        *reinterpret_cast<f32x4*>(&w[x]) = *reinterpret_cast<const f32x4*>(probs + L::prob(h, b * 8 + quad * 2));
                        *(reinterpret_cast<f32x4*>(&w[x]) + 1) = *reinterpret_cast<const f32x4*>(probs + L::prob(h, b * 8 + quad * 2 + 1));
                    }
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint32_t col = wave * (DT * 16) + d * 16; // first of 16 columns
                    Frag<T> f;
                    if constexpr (sizeof(T) == 2) {
                        // a transposing read: lane 4 i + j of 16 points at columns 4 j .. of row i; each lane gets its column's four rows
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t at = value_at[half] + d * 32 + b * (32 * L::kPlaneRow);
                            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_byte*)(tile + at));
                            *(reinterpret_cast<s16x4*>(&f) + half) = v;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float*>(tile + L::at(b * 32 + quad * 8 + i, (col + n) >> 2) + (n & 3) * 4);
                    }
#pragma unroll
                    for (int x = 0; x < HT; ++x) o[x][d] = product16(f, w[x], o[x][d]);
                }
            }
            if (more) {
                if constexpr (L::kBuffers == 2) {
                    settle(now ^ 1, mask);
                    lds_barrier();
                    now ^= 1;
                } else {
                    lds_barrier();
                    find(base + L::kRows);
                    look(base + 2 * L::kRows);
                    bring(0);
                    mask = there;
                    settle(0, mask);
                    lds_barrier();
                }
            }
        }
        // the probabilities' sums over the waves that share a head
        __syncthreads();
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (quad == 0) parts[part * (HT * 16) + ht * 16 + n] = sum;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < HT; ++x) {
            const uint32_t h = x * 16 + n;
            if (h >= heads) continue;
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < L::kParts; ++i) total += parts[i * (HT * 16) + h];
            const float ref = top[x] - kLift<T>; // sums are of 2^(score - ref)
            const uint32_t head = g * a.group + h0 + h;
            const bool whole = c.count == 1;
            const size_t at = static_cast<size_t>(whole ? c.query : c.slot) * a.n_heads + head;
            const float factor = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint32_t col = wave * (DT * 16) + d * 16 + quad * 4; // rows of whole 16-byte words: dv is a multiple of 4
                if (col >= a.dv) continue;
                if (whole) {
                    typedef T Four __attribute__((ext_vector_type(4)));
                    Four f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) f[r] = from_f32<T>(o[x][d][r] * factor);
                    T* out = static_cast<T*>(a.out) + at * a.dv + col;
                    if (a.wide_out) {
                        *reinterpret_cast<Four*>(out) = f;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) out[r] = f[r];
                    }
                } else {
                    *reinterpret_cast<f32x4*>(plan.partial + at * a.dv + col) = o[x][d];
                }
            }
            if (wave == 0 && quad == 0) {
                if (!whole) plan.stats[at] = make_float2(ref, total);
                else if (a.lse) a.lse[at] = total == 0.0f ? -INFINITY : (ref + log2f(total)) * kLn2;
            }
        }
        __syncthreads(); // the next part's queries go where this one's rows were
    } while (walk.next(a, plan, &c));
}

// The chunks of a query joined: out = sum_k 2^(top_k - top) o_k / sum_k 2^(top_k - top) sum_k.  One workgroup per head and query; queries of one chunk are done
// already, queries without rows (no slot is theirs) get their zeros here.  A thread takes W columns of every 256 W / dv-th chunk, so that few long queries
// are not a chain of loads; the threads' parts meet in LDS.
template <typename T, int W> __global__ __launch_bounds__(256) void join_kernel(const AttentionArgs a, const Plan plan) {
    typedef float Cols __attribute__((ext_vector_type(W)));
    __shared__ float weight[256], wide[8];
    __shared__ Cols part[256];
    const uint32_t h = blockIdx.x, i = blockIdx.y, t = threadIdx.x;
    const size_t at = static_cast<size_t>(i) * a.n_heads + h;
    T* out = static_cast<T*>(a.out) + at * a.dv;
    const int32_t* table;
    if (rows_of(a, i, &table) == 0) {
        for (uint32_t col = t; col < a.dv; col += 256) out[col] = from_f32<T>(0.0f);
        if (a.lse && t == 0) a.lse[at] = -INFINITY;
        return;
    }
    const int2 mine = plan.chunks[i];
    if (mine.y == 1) return;
    const uint32_t n = static_cast<uint32_t>(mine.y);
    const float2* stats = plan.stats + static_cast<size_t>(mine.x) * a.n_heads + h;
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t k = t; k < n; k += 256) top = fmaxf(top, stats[static_cast<size_t>(k) * a.n_heads].x);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if ((t & 63) == 0) wide[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wide[0], wide[1]), fmaxf(wide[2], wide[3]));
    const uint32_t cols = a.dv / W; // W divides dv
    const float* partial = plan.partial + (static_cast<size_t>(mine.x) * a.n_heads + h) * a.dv;
    const size_t step = static_cast<size_t>(a.n_heads) * a.dv;
    for (uint32_t base = 0; base < cols; base += 256) { // one turn but for long odd rows
        const uint32_t here = min(256u, cols - base), parts = 256 / here, p = t / here, col = (base + t % here) * W;
        Cols acc = {};
        for (uint32_t first = 0; first < n; first += 256) {
            __syncthreads();
            if (first + t < n) {
                const float2 st = stats[static_cast<size_t>(first + t) * a.n_heads];
                const float w = st.x == -INFINITY ? 0.0f : exp2_fast(st.x - top);
                weight[t] = w;
                if (base == 0) sum += w * st.y;
            }
            __syncthreads();
            const uint32_t some = min(256u, n - first);
            if (p < parts) {
                const float* from = partial + first * step + col;
#pragma unroll 8
                for (uint32_t k = p; k < some; k += parts) acc += weight[k] * *reinterpret_cast<const Cols*>(from + k * step);
            }
        }
        if (base == 0) {
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
            if ((t & 63) == 0) wide[4 + (t >> 6)] = sum;
        }
        part[t] = acc;
        __syncthreads();
        sum = wide[4] + wide[5] + wide[6] + wide[7];
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (t < here) {
            for (uint32_t k = 1; k < parts; ++k) acc += part[t + k * here];
#pragma unroll
            for (int j = 0; j < W; ++j) out[col + j] = from_f32<T>(acc[j] * inv);
        }
    }
    if (a.lse && t == 0) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

int check_attention(const svsx_attention_desc* d, AttentionArgs* a) {
    if (!d) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (d->struct_size != sizeof(svsx_attention_desc))
        return fail(SVSX_INVALID_ARGUMENT, "svsx_attention_desc.struct_size is %zu, expected %zu", d->struct_size, sizeof(svsx_attention_desc));
    if (paged_dtype_size(d->dtype) == 0) return fail(SVSX_INVALID_ARGUMENT, "unsupported row dtype %d (float32, float16, bfloat16)", d->dtype);
    const size_t limit = size_t(1) << 31;
    if (d->n_heads == 0 || d->n_key_heads == 0 || d->n_heads % d->n_key_heads != 0 || d->n_heads > 65535)
        return fail(SVSX_INVALID_ARGUMENT, "n_heads (%zu) must be a multiple of n_key_heads (%zu), and below 65536", d->n_heads, d->n_key_heads);
    if (d->key_dim == 0 || d->value_dim == 0 || d->key_dim > kMaxDim || d->value_dim > kMaxDim)
        return fail(SVSX_INVALID_ARGUMENT, "key_dim (%zu) and value_dim (%zu) must be in [1, %d]", d->key_dim, d->value_dim, kMaxDim);
    if (!d->d_values && d->value_dim > d->key_dim) return fail(SVSX_INVALID_ARGUMENT, "value_dim (%zu) exceeds the key row's %zu columns", d->value_dim, d->key_dim);
    if (d->page_size == 0 || d->page_size >= limit || d->n_pages >= limit || d->n_sequences >= limit || d->max_pages >= limit || d->max_pages * d->page_size >= limit)
        return fail(SVSX_INVALID_ARGUMENT, "page_size must be positive; n_pages, n_sequences and max_pages * page_size must be below 2^31");
    if (d->n_queries > 65535) return fail(SVSX_INVALID_ARGUMENT, "too many queries in one call (%zu, at most 65535)", d->n_queries);
    if (!std::isfinite(d->scale)) return fail(SVSX_INVALID_ARGUMENT, "scale must be finite");
    if (d->n_queries > 0 && (!d->d_queries || !d->d_out)) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (d->n_queries > 0 && d->n_sequences > 0 && (!d->d_lengths || (d->max_pages > 0 && (!d->d_table || (d->n_pages > 0 && !d->d_keys)))))
        return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *a = AttentionArgs{};
    a->queries = d->d_queries;
    a->keys = d->d_keys;
    a->values = d->d_values ? d->d_values : d->d_keys;
    a->table = d->d_table;
    a->lengths = d->d_lengths;
    a->sequences = d->d_sequences;
    a->out = d->d_out;
    a->lse = d->d_lse;
    a->query_stride = d->query_stride;
    a->query_head_stride = d->query_head_stride;
    a->key_page_stride = d->key_page_stride;
    a->key_head_stride = d->key_head_stride;
    a->key_row_stride = d->key_row_stride;
    a->value_page_stride = d->d_values ? d->value_page_stride : d->key_page_stride;
    a->value_head_stride = d->d_values ? d->value_head_stride : d->key_head_stride;
    a->value_row_stride = d->d_values ? d->value_row_stride : d->key_row_stride;
    a->table_stride = d->table_stride;
    a->n_queries = static_cast<uint32_t>(d->n_queries);
    a->n_heads = static_cast<uint32_t>(d->n_heads);
    a->n_key_heads = static_cast<uint32_t>(d->n_key_heads);
    a->group = static_cast<uint32_t>(d->n_heads / d->n_key_heads);
    a->dk = static_cast<uint32_t>(d->key_dim);
    a->dv = static_cast<uint32_t>(d->value_dim);
    a->n_pages = static_cast<uint32_t>(d->n_pages);
    a->page_size = static_cast<uint32_t>(d->page_size);
    a->n_sequences = static_cast<uint32_t>(d->n_sequences);
    a->max_pages = static_cast<uint32_t>(d->max_pages);
    a->scale = d->scale;
    a->shared = d->d_values == nullptr;
    const size_t es = paged_dtype_size(d->dtype);
    a->wide_out = d->value_dim % 8 == 0 && (reinterpret_cast<size_t>(d->d_out) & 15) == 0;
    a->wide_queries = d->key_dim % 8 == 0 && ((reinterpret_cast<size_t>(d->d_queries) | d->query_stride * es | d->query_head_stride * es) & 15) == 0;
    return SVSX_SUCCESS;
}

// How a call is answered; decided from sizes, types, strides and addresses alone.
struct Route {
    bool rows, group, few; // many heads over shared rows, or heads that share a key head, on the matrix units; few rows, one head; else one workgroup per head
    bool wide, page8;
    int ks, vb, ht;
    uint32_t workers, unit, y;
    size_t stats_at, chunks_at, bytes;
};

// Workgroups that are resident at once, on 256 compute units: all rows are cut into as many equal runs.
constexpr uint32_t kUnits = 256;

Route route_of(const AttentionArgs& a, size_t es) {
    Route r = {};
    auto aligned = [&](std::initializer_list<size_t> strides, const void* p) {
        size_t all = reinterpret_cast<size_t>(p);
        for (size_t x : strides) all |= x * es;
        return all % 16 == 0;
    };
    r.wide = a.dk % 8 == 0 && a.dv % 8 == 0 && aligned({a.key_page_stride, a.key_head_stride, a.key_row_stride}, a.keys) &&
             aligned({a.value_page_stride, a.value_head_stride, a.value_row_stride}, a.values);
    // Shared rows go through LDS where more than 16 heads read them, and where they are so long that the other kernel reads them twice (32 queries of 4096 float16 rows: 16 heads,
    // 128 columns 25 us either way, 256 columns 26 us against 45; 32 heads 27 against 29, 29 against 52; 8 heads, 128 columns 24 against 22).
    r.rows = a.shared && r.wide && a.dk <= 576 && a.dv <= 512 && (a.group > 16 || a.dk > 128);
    const uint64_t most = static_cast<uint64_t>(a.max_pages) * a.page_size; // rows that a query can have
    const uint64_t items = static_cast<uint64_t>(a.n_queries) * a.n_key_heads; // one wave each
    r.few = a.group == 1 && most <= kFewRows && items >= kFewItems && items <= 1u << 25 && a.dk <= 256 && a.dv <= 256; // a grid has fewer than 2^32 threads
    if (r.few) {
        r.rows = false;
        return r;
    }
    r.group = !r.rows && a.dk <= 256 && a.dv <= 256;
    if (!r.rows && !r.group) return r;
    if (r.rows) {
        r.ks = a.dk <= 320 && a.dv <= 256 ? 10 : 18;
        // 32 sequences of 4096 bfloat16 rows, 576 columns, by 16, 32 or 64 heads a workgroup: 16 heads 36, 38, 44 us; 32 heads 48, 41, 46; 64 heads 79, 59, 54; 128 heads 136, 94, 79.
        // float32 queries of 16 heads fill the registers.
        r.ht = a.group <= 16 || es == 4 ? 1 : a.group <= 32 ? 2 : 4;
        r.unit = 64;
        r.y = a.n_key_heads * ((a.group + r.ht * 16 - 1) / (r.ht * 16));
    } else {
        r.page8 = a.page_size % 8 == 0;
        r.vb = a.dv > 128 || a.dk > 128 ? 2 : 1;
        r.ks = !r.wide ? (r.vb == 2 ? 8 : 4) : a.dk > 192 ? 8 : a.dk > 128 || r.vb == 2 ? 6 : a.dk > 96 ? 4 : a.dk > 64 ? 3 : 2;
        r.unit = kChunkUnit;
        r.y = a.n_key_heads * ((a.group + 15) / 16);
    }
    // One workgroup a query where queries alone fill the machine several times over, where no query can have more rows than one unit, or where the sum of all units
    // might not fit 32 bits.  32 heads on 8 of 128 float16 columns, one workgroup a query against equal runs: 512 queries of 1000 rows 305 and 385 us, of lengths up to 1000 204 and 231; but 256
    // queries, two of them of 4000 rows and the others below 500, 149 and 86.
    const uint32_t resident = kUnits * (r.rows ? 1 : r.vb == 2 || es == 4 ? 2 : 3);
    const uint64_t groups = static_cast<uint64_t>(a.n_queries) * r.y, units = (most + r.unit - 1) / r.unit;
    if (groups >= 4 * resident || units <= 1 || units * a.n_queries >= (1ull << 32)) return r;
    r.workers = static_cast<uint32_t>(std::min<uint64_t>(std::max(1u, resident / r.y), a.n_queries * units));
    const size_t parts = (static_cast<size_t>(r.workers) + a.n_queries) * a.n_heads;
    r.stats_at = (parts * a.dv * 4 + 15) / 16 * 16;
    r.chunks_at = r.stats_at + parts * 8;
    r.bytes = r.chunks_at + static_cast<size_t>(a.n_queries) * 8;
    return r;
}

template <typename T, int KS, int HT> hipError_t launch_rows(const AttentionArgs& a, const Plan& plan, const Route& r, hipStream_t stream) {
    typedef RowsLayout<T, KS, HT> L;
    static std::atomic<uint64_t> granted{0};
    if (const hipError_t e = grant_lds(reinterpret_cast<const void*>(attend_rows_kernel<T, KS, HT>), L::kBytes, &granted); e != hipSuccess) return e;
    hipLaunchKernelGGL((attend_rows_kernel<T, KS, HT>), dim3(r.workers ? r.workers : a.n_queries, r.y), dim3(L::kThreads), L::kBytes, stream, a, plan, divider(a.page_size));
    return hipGetLastError();
}

template <typename T> hipError_t launch_rows(const AttentionArgs& a, const Plan& plan, const Route& r, hipStream_t stream) {
    if (r.ks == 10) {
        if (r.ht == 1) return launch_rows<T, 10, 1>(a, plan, r, stream);
        if constexpr (sizeof(T) == 2) return r.ht == 2 ? launch_rows<T, 10, 2>(a, plan, r, stream) : launch_rows<T, 10, 4>(a, plan, r, stream);
    } else {
        if (r.ht == 1) return launch_rows<T, 18, 1>(a, plan, r, stream);
        if constexpr (sizeof(T) == 2) return r.ht == 2 ? launch_rows<T, 18, 2>(a, plan, r, stream) : launch_rows<T, 18, 4>(a, plan, r, stream);
    }
    return hipErrorInvalidValue;
}

template <typename T> hipError_t launch_split(const AttentionArgs& a, const Route& r, void* workspace, hipStream_t stream) {
    Plan plan = {};
    plan.workers = r.workers;
    plan.unit = r.unit;
    if (r.workers) {
        char* base = static_cast<char*>(workspace);
        plan.partial = reinterpret_cast<float*>(base);
        plan.stats = reinterpret_cast<float2*>(base + r.stats_at);
        plan.chunks = reinterpret_cast<int2*>(base + r.chunks_at);
    }
    typedef void (*Kernel)(const AttentionArgs, const Plan, const Divider);
    Kernel kernel = nullptr;
#define SVSX_GROUP(KS, VB, WIDE) \
    if (r.ks == KS && r.vb == VB && r.wide == WIDE) kernel = r.page8 ? attend_group_kernel<T, KS, VB, WIDE, true> : attend_group_kernel<T, KS, VB, WIDE, false>;
    SVSX_GROUP(2, 1, true)
    SVSX_GROUP(3, 1, true)
    SVSX_GROUP(4, 1, true)
    SVSX_GROUP(6, 2, true)
    SVSX_GROUP(8, 2, true)
    SVSX_GROUP(4, 1, false)
    SVSX_GROUP(8, 2, false)
#undef SVSX_GROUP
    if (r.rows) {
        const hipError_t e = launch_rows<T>(a, plan, r, stream);
        if (e != hipSuccess) return e;
    } else {
        if (!kernel) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kernel, dim3(r.workers ? r.workers : a.n_queries, r.y), dim3(256), 0, stream, a, plan, divider(a.page_size));
    }
    if (r.workers) hipLaunchKernelGGL((a.dv % 4 == 0 ? join_kernel<T, 4> : join_kernel<T, 1>), dim3(a.n_heads, a.n_queries), dim3(256), 0, stream, a, plan);
    return hipGetLastError();
}

template <typename T> hipError_t launch_attention(const AttentionArgs& a, const Route& r, void* workspace, hipStream_t stream) {
    if (r.few) {
        const bool narrow = a.dk <= 128 && a.dv <= 128;
        typedef void (*Kernel)(const AttentionArgs, const Divider);
        Kernel kernel;
        if (narrow) kernel = r.wide ? attend_few_kernel<T, 8, true> : attend_few_kernel<T, 8, false>;
        else kernel = r.wide ? attend_few_kernel<T, 16, true> : attend_few_kernel<T, 16, false>;
        hipLaunchKernelGGL(kernel, dim3((a.n_queries * a.n_key_heads + 3) / 4), dim3(256), 0, stream, a, divider(a.page_size));
        return hipGetLastError();
    }
    if (r.rows || r.group) return launch_split<T>(a, r, workspace, stream);
    hipLaunchKernelGGL(attend_head_kernel<T>, dim3(a.n_heads, a.n_queries), dim3(256), 0, stream, a);
    return hipGetLastError();
}

} // namespace
} // namespace svsx

extern "C" {

int svsx_paged_attention_workspace(const svsx_attention_desc* desc, size_t* bytes) {
    AttentionArgs a;
    if (const int rc = check_attention(desc, &a)) return rc;
    if (!bytes) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *bytes = a.n_queries ? route_of(a, paged_dtype_size(desc->dtype)).bytes : 0;
    return SVSX_SUCCESS;
}

int svsx_paged_attention_device(const svsx_attention_desc* desc, void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    AttentionArgs a;
    if (const int rc = check_attention(desc, &a)) return rc;
    if (a.n_queries == 0) return SVSX_SUCCESS;
    const Route r = route_of(a, paged_dtype_size(desc->dtype));
    if (r.bytes > 0 && (!d_workspace || workspace_bytes < r.bytes || reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0))
        return fail(SVSX_INVALID_ARGUMENT, "a workspace of %zu bytes, aligned to 16, is needed", r.bytes);
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = desc->dtype == SVSX_F32   ? launch_attention<float>(a, r, d_workspace, s)
                         : desc->dtype == SVSX_F16 ? launch_attention<_Float16>(a, r, d_workspace, s)
                                                   : launch_attention<bf16_t>(a, r, d_workspace, s);
    return e == hipSuccess ? SVSX_SUCCESS : fail(SVSX_RUNTIME_ERROR, "attention launch failed: %s", hipGetErrorString(e));
}

} // extern "C"
