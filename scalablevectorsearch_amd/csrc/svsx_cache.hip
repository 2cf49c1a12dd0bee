// svsx_cache.hip -- a paged cache of rows and its page operations (include/svsx.h: svsx_cache_*).
//
// The cache is plain arrays in HBM: pages of rows [layer][page][head][row in page][dim], a table of pages per sequence, the sequences' lengths, and one
// reference count per page.  Every operation runs on the device from those arrays alone, in stream order and without a host round trip, so a
// serving loop can capture it.  The rule that makes results reproducible: an operation that needs pages takes the LOWEST free ones, in the order of its
// entries.  Shared pages are always full (a fork copies a partly filled last page), so a row is never written to a page that two sequences hold.
//
// An operation is a planning kernel -- ONE workgroup (8 to 10 us, a chain of dependent loads), because ranks among the free pages are a running count over all of them -- and, where rows move, a
// second kernel that fills the machine with copies.  The planner's time grows with the pool, 16384 pages a step: 64 sequences that take a page each and give it back, with all pages but the last 200
// held: 2000 pages 13 us, 20000 15, 200000 34, a million 121; compaction of nothing 11, 22, 145, 716.
#include "svsx_host.h"
#include "svsx_paged.h"
#include <initializer_list>

namespace svsx {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kMaxSequences = 4096;                      // a claim, a running count and a length per sequence in the planner's LDS (48 KB, and 8 of pages)
constexpr int kPerThread = kMaxSequences / kPlanThreads; // entries a planner thread scans
constexpr int kNear = 2048;                              // pages by rank that stay in LDS; what is beyond goes through the workspace
constexpr int kPagesPerThread = 16;                      // reference counts a planner thread reads per step (four 16-byte loads in flight)

struct CacheArgs {
    unsigned char* keys;
    unsigned char* values;
    int32_t* table;
    int32_t* lengths;
    int32_t* refs;
    int32_t* failures;
    uint32_t n_layers, n_pages, n_heads, page_size, n_sequences, columns;
    size_t key_row_bytes, value_row_bytes; // one row of one head
};

// what the planning kernel hands to the copying kernel
struct PlanSpace {
    int32_t* start; // per entry: length before the call, -1 = refused
    int32_t* from;  // per new page, by rank: page copied from (-1: none), page copied to, rows
    int32_t* to;
    int32_t* rows;
    int32_t* count; // [0] pages by rank
};

__device__ __forceinline__ int wave_inclusive(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(v, off);
        if (lane >= off) v += u;
    }
    return v;
}

// exclusive running count over the workgroup's threads; *total = sum.  Two barriers; `waves` is reused by the next call.
__device__ __forceinline__ int block_exclusive(int v, int* waves, int* total) {
    const int incl = wave_inclusive(v), wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) waves[wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const int x = waves[w];
        before += w < wave ? x : 0;
        all += x;
    }
    *total = all;
    return before + incl - v;
}

// the reference counts of this thread's kPagesPerThread pages from `first` on; beyond the pool: `beyond`
__device__ __forceinline__ void load_refs(const CacheArgs& a, uint32_t first, int beyond, int (&r)[kPagesPerThread]) {
    if (first + kPagesPerThread <= a.n_pages && (reinterpret_cast<uintptr_t>(a.refs) & 15) == 0) {
        const int4* p = reinterpret_cast<const int4*>(a.refs + first);
#pragma unroll
        for (int i = 0; i < kPagesPerThread / 4; ++i) {
            const int4 v = p[i];
            r[4 * i] = v.x;
            r[4 * i + 1] = v.y;
            r[4 * i + 2] = v.z;
            r[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) r[i] = first + i < a.n_pages ? a.refs[first + i] : beyond;
    }
}

struct PlanShared {
    int claim[kMaxSequences]; // which entry of the call has this sequence for its own (the first that names it)
    int incl[kMaxSequences];  // running count of the pages that the entries up to this one need
    int length[kMaxSequences]; // of an entry's sequence before the call; -1 = refused
    int list[kNear];          // the first pages by rank
    int waves[kPlanWaves];
    int bad, refused;
};

// the `want` lowest free pages to sh.list[], from kNear on to list[]; returns how many there are (at most want)
__device__ __forceinline__ int lowest_free(const CacheArgs& a, int want, int32_t* list, PlanShared& sh) {
    int found = 0;
    for (uint32_t base = 0; base < a.n_pages && found < want; base += kPlanThreads * kPagesPerThread) {
        const uint32_t first = base + threadIdx.x * kPagesPerThread;
        int r[kPagesPerThread], mine = 0, total;
        load_refs(a, first, 1, r);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) mine += r[i] == 0;
        int rank = found + block_exclusive(mine, sh.waves, &total);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) {
            if (r[i] == 0) {
                if (rank < want) {
                    if (rank < kNear) sh.list[rank] = static_cast<int32_t>(first + i);
                    else list[rank] = static_cast<int32_t>(first + i);
                }
                ++rank;
            }
        }
        found += total;
    }
    __syncthreads();
    return found < want ? found : want;
}

// sh.incl[] from each entry's need; returns the sum.  Needs are at most the table's columns, so the sum stays below 2^31 (checked on the host).
__device__ __forceinline__ int scan_needs(PlanShared& sh, const int (&need)[kPerThread]) {
    int mine = 0, total;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) mine += need[e];
    int run = block_exclusive(mine, sh.waves, &total);
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        run += need[e];
        sh.incl[threadIdx.x * kPerThread + e] = run;
    }
    __syncthreads();
    return total;
}

// the entry whose pages include the one of this rank: the first with incl > rank
__device__ __forceinline__ int entry_of(const PlanShared& sh, int n, int rank) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sh.incl[mid] > rank) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ void claim_sequences(const CacheArgs& a, PlanShared& sh, const int32_t* seqs, int n) {
    for (uint32_t s = threadIdx.x; s < a.n_sequences; s += kPlanThreads) sh.claim[s] = n;
    if (threadIdx.x == 0) sh.bad = sh.refused = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t s = seqs[i];
        if (s >= 0 && static_cast<uint32_t>(s) < a.n_sequences) atomicMin(&sh.claim[s], i);
    }
    __syncthreads();
}

// The slot (page * page_size + row in page) of new row t; -1 where its sequence was refused (start -1) or no entry has it.
__device__ __forceinline__ int64_t slot_of(const CacheArgs& a, const int32_t* seqs, const int32_t* offsets, int n, int t, const int32_t* start) {
    if (n == 0) return -1;
    int lo = 0, hi = n; // the last entry whose rows begin at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int32_t old = start[lo];
    if (old < 0 || t < offsets[lo] || t >= offsets[lo + 1]) return -1;
    const uint32_t at = static_cast<uint32_t>(old) + static_cast<uint32_t>(t - offsets[lo]);
    const int32_t page = a.table[static_cast<size_t>(seqs[lo]) * a.columns + at / a.page_size];
    return page >= 0 && static_cast<uint32_t>(page) < a.n_pages ? static_cast<int64_t>(page) * a.page_size + at % a.page_size : -1;
}

// Sequence seqs[i] grows by offsets[i + 1] - offsets[i] rows.
__global__ __launch_bounds__(kPlanThreads) void extend_plan_kernel(const CacheArgs a, const int32_t* seqs, const int32_t* offsets, int n, int n_tokens, PlanSpace ws, int64_t* slots) {
    __shared__ PlanShared sh;
    claim_sequences(a, sh, seqs, n);
    // offsets that run backwards or out of the call's rows refuse the call: no entry could be told from another's rows
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (offsets[i] < 0 || offsets[i + 1] < offsets[i] || offsets[i + 1] > n_tokens) sh.bad = 1;
    __syncthreads();
    const bool bad = sh.bad != 0;
    int need[kPerThread], old[kPerThread], grown[kPerThread];
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int i = threadIdx.x * kPerThread + e;
        need[e] = 0;
        old[e] = -1;
        grown[e] = 0;
        if (i >= n || bad) continue;
        const int32_t s = seqs[i];
        if (s < 0 || static_cast<uint32_t>(s) >= a.n_sequences || sh.claim[s] != i) continue;
        const uint32_t len = static_cast<uint32_t>(a.lengths[s]), count = static_cast<uint32_t>(offsets[i + 1] - offsets[i]);
        const uint64_t pages = (static_cast<uint64_t>(len) + count + a.page_size - 1) / a.page_size;
        if (pages > a.columns) continue;
        need[e] = static_cast<int>(pages) - static_cast<int>((len + a.page_size - 1) / a.page_size);
        old[e] = static_cast<int>(len);
        grown[e] = static_cast<int>(len + count);
        sh.length[i] = old[e];
    }
    const int total = scan_needs(sh, need);
    const int have = lowest_free(a, total, ws.to, sh);
    for (int rank = threadIdx.x; rank < have; rank += kPlanThreads) {
        const int i = entry_of(sh, n, rank);
        if (sh.incl[i] > have) continue; // the first entry that does not fit
        const int32_t s = seqs[i], page = rank < kNear ? sh.list[rank] : ws.to[rank];
        const int first = i == 0 ? 0 : sh.incl[i - 1];
        const uint32_t column = (static_cast<uint32_t>(sh.length[i]) + a.page_size - 1) / a.page_size + (rank - first);
        a.table[static_cast<size_t>(s) * a.columns + column] = page;
        a.refs[page] = 1;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int i = threadIdx.x * kPerThread + e;
        if (i >= n) continue;
        const bool served = old[e] >= 0 && (need[e] == 0 || sh.incl[i] <= have);
        sh.length[i] = served ? old[e] : -1;
        if (!slots) ws.start[i] = sh.length[i];
        if (served) a.lengths[seqs[i]] = grown[e];
        else atomicAdd(&sh.refused, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.refused) atomicAdd(a.failures, sh.refused);
    if (slots)
        for (int t = threadIdx.x; t < n_tokens; t += kPlanThreads) slots[t] = slot_of(a, seqs, offsets, n, t, sh.length);
}

// The slots of a call of many rows.
__global__ __launch_bounds__(256) void slots_kernel(const CacheArgs a, const int32_t* seqs, const int32_t* offsets, int n, int n_tokens, const int32_t* start, int64_t* slots) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < n_tokens) slots[t] = slot_of(a, seqs, offsets, n, t, start);
}

// Sequence targets[i], empty until now, becomes sources[i]: sharing its full pages (share) or with pages of its own.
__global__ __launch_bounds__(kPlanThreads) void copy_plan_kernel(const CacheArgs a, const int32_t* sources, const int32_t* targets, int n, int share, PlanSpace ws) {
    __shared__ PlanShared sh;
    claim_sequences(a, sh, targets, n);
    int need[kPerThread], len[kPerThread];
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int i = threadIdx.x * kPerThread + e;
        need[e] = 0;
        len[e] = -1;
        if (i >= n) continue;
        const int32_t s = sources[i], t = targets[i];
        if (s < 0 || t < 0 || static_cast<uint32_t>(s) >= a.n_sequences || static_cast<uint32_t>(t) >= a.n_sequences) continue;
        if (sh.claim[t] != i || sh.claim[s] != n || a.lengths[t] != 0) continue; // a target twice, a source that is a target too, a target that holds rows
        len[e] = a.lengths[s];
        const uint32_t l = static_cast<uint32_t>(len[e]);
        if (len[e] < 0 || static_cast<uint64_t>(l) > static_cast<uint64_t>(a.columns) * a.page_size) { // no length that this cache can hold
            len[e] = -1;
            continue;
        }
        need[e] = static_cast<int>(share ? (l % a.page_size != 0) : (l + a.page_size - 1) / a.page_size);
        sh.length[i] = len[e];
    }
    const int total = scan_needs(sh, need);
    const int have = lowest_free(a, total, ws.to, sh);
    for (int rank = threadIdx.x; rank < have; rank += kPlanThreads) {
        const int i = entry_of(sh, n, rank);
        int32_t from = -1;
        if (sh.incl[i] <= have) {
            const int32_t s = sources[i], page = rank < kNear ? sh.list[rank] : ws.to[rank];
            if (rank < kNear) ws.to[rank] = page;
            const uint32_t l = static_cast<uint32_t>(sh.length[i]), first = i == 0 ? 0 : sh.incl[i - 1];
            const uint32_t column = (share ? l / a.page_size : 0) + (rank - first);
            from = a.table[static_cast<size_t>(s) * a.columns + column];
            a.table[static_cast<size_t>(targets[i]) * a.columns + column] = page;
            a.refs[page] = 1;
            const uint32_t left = l - column * a.page_size;
            ws.rows[rank] = static_cast<int32_t>(left < a.page_size ? left : a.page_size);
        }
        ws.from[rank] = from;
    }
    if (threadIdx.x == 0) ws.count[0] = have;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int i = threadIdx.x * kPerThread + e;
        if (i >= n) continue;
        const bool served = len[e] >= 0 && (need[e] == 0 || sh.incl[i] <= have);
        ws.start[i] = served ? len[e] : -1;
        if (served) a.lengths[targets[i]] = len[e]; // a target is no source: nobody reads this length here
        else atomicAdd(&sh.refused, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.refused) atomicAdd(a.failures, sh.refused);
}

// Used pages from U = the number of used pages on go, in order, to the free pages below U, in order.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const CacheArgs a, PlanSpace ws, int32_t* moved) {
    __shared__ PlanShared sh;
    int used = 0, r[kPagesPerThread];
    for (uint32_t base = 0; base < a.n_pages; base += kPlanThreads * kPagesPerThread) {
        load_refs(a, base + threadIdx.x * kPagesPerThread, 0, r);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) used += r[i] > 0;
    }
    int U;
    block_exclusive(used, sh.waves, &U);
    int holes = 0, movers = 0;
    for (uint32_t base = 0; base < a.n_pages; base += kPlanThreads * kPagesPerThread) {
        const uint32_t first = base + threadIdx.x * kPagesPerThread;
        load_refs(a, first, 0, r);
        int h = 0, m = 0, all_h, all_m;
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) {
            const bool below = first + i < static_cast<uint32_t>(U);
            h += below && r[i] <= 0;
            m += !below && r[i] > 0;
        }
        int at_h = holes + block_exclusive(h, sh.waves, &all_h), at_m = movers + block_exclusive(m, sh.waves, &all_m);
#pragma unroll
        for (int i = 0; i < kPagesPerThread; ++i) {
            const uint32_t p = first + i;
            if (p >= a.n_pages) continue;
            const bool below = p < static_cast<uint32_t>(U);
            if (below && r[i] <= 0) ws.to[at_h++] = static_cast<int32_t>(p);
            if (!below && r[i] > 0) ws.from[at_m++] = static_cast<int32_t>(p);
            moved[p] = r[i] > 0 ? static_cast<int32_t>(p) : -1;
        }
        holes += all_h;
        movers += all_m;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPlanThreads) { // as many holes as movers: both are U less the used pages below U
        const int32_t from = ws.from[k], to = ws.to[k];
        moved[from] = to;
        a.refs[to] = a.refs[from];
        a.refs[from] = 0;
        ws.rows[k] = static_cast<int32_t>(a.page_size);
    }
    if (threadIdx.x == 0) ws.count[0] = movers;
}

// One wave copies `bytes` (a multiple of sizeof(W)) from one place to another that does not overlap it.
template <typename W> __device__ __forceinline__ void wave_copy(const unsigned char* src, unsigned char* dst, size_t bytes) {
    const W* s = reinterpret_cast<const W*>(src);
    W* d = reinterpret_cast<W*>(dst);
    const size_t n = bytes / sizeof(W);
    size_t i = threadIdx.x & 63;
    for (; i + 192 < n; i += 256) { // four loads in flight per lane
        const W v0 = s[i], v1 = s[i + 64], v2 = s[i + 128], v3 = s[i + 192];
        d[i] = v0;
        d[i + 64] = v1;
        d[i + 128] = v2;
        d[i + 192] = v3;
    }
    for (; i < n; i += 64) d[i] = s[i];
}

// Row data of the planned pages, one wave per (page, layer, head, keys or values): rows of one head in one page are contiguous.  The waves of a fixed
// grid share the units out in turn, because only the device knows how many pages there are.  16 sequences of 1019 rows, 2 layers, copied (267 MB read and written): 5.9 TB/s.
template <typename W> __device__ __forceinline__ void move_pages(const CacheArgs& a, const PlanSpace& ws) {
    const uint32_t kinds = a.value_row_bytes ? 2u : 1u;
    const uint64_t per_page = static_cast<uint64_t>(a.n_layers) * a.n_heads * kinds, units = per_page * static_cast<uint32_t>(ws.count[0]);
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += static_cast<uint64_t>(gridDim.x) * 4) {
        const uint32_t k = static_cast<uint32_t>(u / per_page), in_page = static_cast<uint32_t>(u % per_page);
        const uint32_t kind = in_page % kinds, head = in_page / kinds % a.n_heads, layer = in_page / kinds / a.n_heads;
        const int32_t from = ws.from[k], to = ws.to[k];
        if (from < 0 || static_cast<uint32_t>(from) >= a.n_pages) continue;
        const size_t row = kind ? a.value_row_bytes : a.key_row_bytes, block = row * a.page_size;
        unsigned char* base = kind ? a.values : a.keys;
        const size_t page0 = static_cast<size_t>(layer) * a.n_pages;
        wave_copy<W>(base + ((page0 + from) * a.n_heads + head) * block, base + ((page0 + to) * a.n_heads + head) * block, row * ws.rows[k]);
    }
}

template <typename W> __global__ __launch_bounds__(256) void copy_pages_kernel(const CacheArgs a, const int32_t* sources, const int32_t* targets, int n, int share, PlanSpace ws) {
    if (share) {
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
            if (ws.start[i] < 0) continue;
            const uint32_t whole = static_cast<uint32_t>(ws.start[i]) / a.page_size;
            const int32_t* from = a.table + static_cast<size_t>(sources[i]) * a.columns;
            int32_t* to = a.table + static_cast<size_t>(targets[i]) * a.columns;
            for (uint32_t c = threadIdx.x; c < whole; c += 256) {
                const int32_t page = from[c];
                to[c] = page;
                if (page >= 0 && static_cast<uint32_t>(page) < a.n_pages) atomicAdd(&a.refs[page], 1);
            }
        }
    }
    move_pages<W>(a, ws);
}

template <typename W> __global__ __launch_bounds__(256) void compact_pages_kernel(const CacheArgs a, const int32_t* moved, PlanSpace ws) {
    for (uint32_t s = blockIdx.x; s < a.n_sequences; s += gridDim.x) {
        const uint32_t pages = (static_cast<uint32_t>(a.lengths[s]) + a.page_size - 1) / a.page_size;
        int32_t* row = a.table + static_cast<size_t>(s) * a.columns;
        for (uint32_t c = threadIdx.x; c < pages && c < a.columns; c += 256) {
            const int32_t page = row[c];
            if (page >= 0 && static_cast<uint32_t>(page) < a.n_pages) row[c] = moved[page];
        }
    }
    move_pages<W>(a, ws);
}

// The sequence gives up its pages.  Each table entry is exchanged for -1, so a sequence that is named twice gives each page up once.
__global__ __launch_bounds__(256) void free_kernel(const CacheArgs a, const int32_t* seqs, int n) {
    __shared__ int length;
    const int32_t s = seqs[blockIdx.x];
    if (s < 0 || static_cast<uint32_t>(s) >= a.n_sequences) {
        if (threadIdx.x == 0) atomicAdd(a.failures, 1);
        return;
    }
    if (threadIdx.x == 0) length = atomicExch(&a.lengths[s], 0);
    __syncthreads();
    const uint32_t pages = (static_cast<uint32_t>(length) + a.page_size - 1) / a.page_size;
    int32_t* row = a.table + static_cast<size_t>(s) * a.columns;
    for (uint32_t c = threadIdx.x; c < pages && c < a.columns; c += 256) {
        const int32_t page = atomicExch(&row[c], -1);
        if (page >= 0 && static_cast<uint32_t>(page) < a.n_pages) atomicSub(&a.refs[page], 1);
    }
}

struct WriteArgs {
    const int64_t* slots;
    const unsigned char* src[2]; // keys, values
    unsigned char* dst[2];       // this layer's pages
    size_t token_bytes[2], head_bytes[2];
    uint32_t row_words[2];
    uint32_t n_tokens, n_heads, page_size, n_pages;
};

// One thread per word of a row (16 bytes where rows allow it), several words a thread where a grid, which has fewer than 2^32 threads, would not hold them.  16381 rows of 8 heads, keys and values, float32: 49 us, 5.5 TB/s read and written; 128 rows: 2.9 us.
template <typename W> __global__ __launch_bounds__(256) void write_kernel(const WriteArgs a) {
    const uint32_t kind = blockIdx.y, words = a.row_words[kind], per_token = words * a.n_heads;
    const uint64_t all = static_cast<uint64_t>(a.n_tokens) * per_token;
    for (uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; at < all; at += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint32_t token = static_cast<uint32_t>(at / per_token), in_token = static_cast<uint32_t>(at % per_token);
        const int64_t slot = a.slots[token];
        if (slot < 0 || slot >= static_cast<int64_t>(a.n_pages) * a.page_size) continue;
        const uint32_t head = in_token / words, word = in_token % words;
        const size_t page = static_cast<size_t>(slot) / a.page_size, row = static_cast<size_t>(slot) % a.page_size;
        const W* s = reinterpret_cast<const W*>(a.src[kind] + token * a.token_bytes[kind] + head * a.head_bytes[kind]);
        W* d = reinterpret_cast<W*>(a.dst[kind]) + ((page * a.n_heads + head) * a.page_size + row) * words;
        d[word] = s[word];
    }
}

int check_cache(const svsx_cache_desc* d, CacheArgs* a) {
    if (!d) return fail(SVSX_NOT_INITIALIZED, "Cache not initialized");
    if (d->struct_size != sizeof(svsx_cache_desc)) return fail(SVSX_INVALID_ARGUMENT, "svsx_cache_desc.struct_size is %zu, expected %zu", d->struct_size, sizeof(svsx_cache_desc));
    const size_t es = paged_dtype_size(d->dtype);
    if (es == 0) return fail(SVSX_INVALID_ARGUMENT, "unsupported row dtype %d (float32, float16, bfloat16)", d->dtype);
    const size_t limit = size_t(1) << 31;
    if (d->n_layers == 0 || d->n_pages == 0 || d->n_heads == 0 || d->page_size == 0 || d->key_dim == 0) return fail(SVSX_INVALID_ARGUMENT, "empty cache");
    if (d->n_pages >= limit || d->n_layers >= limit || d->n_heads >= limit || d->page_size >= limit || d->key_dim >= limit || d->value_dim >= limit)
        return fail(SVSX_INVALID_ARGUMENT, "a size of the cache exceeds 2^31 - 1");
    if (d->n_sequences == 0 || d->n_sequences > kMaxSequences) return fail(SVSX_INVALID_ARGUMENT, "n_sequences must be in [1, %d]", kMaxSequences);
    if (d->max_pages == 0 || d->max_pages >= limit || d->max_pages * d->page_size >= limit) return fail(SVSX_INVALID_ARGUMENT, "max_pages * page_size must be in [1, 2^31)");
    if (d->max_pages * d->n_sequences >= limit) return fail(SVSX_INVALID_ARGUMENT, "max_pages * n_sequences must be below 2^31");
    if (!d->d_keys || !d->d_table || !d->d_lengths || !d->d_refs || !d->d_failures) return fail(SVSX_INVALID_ARGUMENT, "null cache array");
    if ((d->value_dim != 0) != (d->d_values != nullptr)) return fail(SVSX_INVALID_ARGUMENT, "value_dim and d_values do not agree");
    a->keys = static_cast<unsigned char*>(d->d_keys);
    a->values = static_cast<unsigned char*>(d->d_values);
    a->table = d->d_table;
    a->lengths = d->d_lengths;
    a->refs = d->d_refs;
    a->failures = d->d_failures;
    a->n_layers = static_cast<uint32_t>(d->n_layers);
    a->n_pages = static_cast<uint32_t>(d->n_pages);
    a->n_heads = static_cast<uint32_t>(d->n_heads);
    a->page_size = static_cast<uint32_t>(d->page_size);
    a->n_sequences = static_cast<uint32_t>(d->n_sequences);
    a->columns = static_cast<uint32_t>(d->max_pages);
    a->key_row_bytes = d->key_dim * es;
    a->value_row_bytes = d->value_dim * es;
    return SVSX_SUCCESS;
}

int check_entries(size_t n, const void* a, const void* b) {
    if (n > kMaxSequences) return fail(SVSX_INVALID_ARGUMENT, "too many sequences in one call (%zu, at most %d)", n, kMaxSequences);
    if (n > 0 && (!a || !b)) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    return SVSX_SUCCESS;
}

size_t workspace_bytes(const CacheArgs& a, size_t n) { return 4 * (n + 3 * static_cast<size_t>(a.n_pages) + 1); }

int carve(const CacheArgs& a, size_t n, void* ws, size_t bytes, PlanSpace* p) {
    if (!ws || bytes < workspace_bytes(a, n)) return fail(SVSX_INVALID_ARGUMENT, "workspace of %zu bytes, %zu needed", bytes, workspace_bytes(a, n));
    if (reinterpret_cast<uintptr_t>(ws) & 3) return fail(SVSX_INVALID_ARGUMENT, "workspace must be aligned to 4 bytes");
    p->count = static_cast<int32_t*>(ws);
    p->start = p->count + 1;
    p->from = p->start + n;
    p->to = p->from + a.n_pages;
    p->rows = p->to + a.n_pages;
    return SVSX_SUCCESS;
}

// the widest word that divides every row and address
size_t word_of(std::initializer_list<size_t> all) {
    size_t bits = 16;
    for (size_t x : all) bits |= x;
    return bits & (~bits + 1);
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SVSX_SUCCESS : fail(SVSX_RUNTIME_ERROR, "%s launch failed: %s", what, hipGetErrorString(e));
}

size_t page_word(const CacheArgs& a) {
    return word_of({reinterpret_cast<size_t>(a.keys), reinterpret_cast<size_t>(a.values), a.key_row_bytes, a.value_row_bytes});
}
constexpr int kMoveBlocks = 2048; // eight workgroups per compute unit
constexpr size_t kWriteBlocks = size_t(1) << 20; // 2^28 threads

} // namespace
} // namespace svsx

extern "C" {

int svsx_cache_workspace(const svsx_cache_desc* desc, size_t n, size_t* bytes) {
    CacheArgs a;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (const int rc = check_entries(n, bytes, bytes)) return rc;
    if (!bytes) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *bytes = workspace_bytes(a, n);
    return SVSX_SUCCESS;
}

int svsx_cache_extend_device(const svsx_cache_desc* desc, const int32_t* d_sequences, const int32_t* d_offsets, size_t n, size_t n_tokens, int64_t* d_slots,
                             void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    CacheArgs a;
    PlanSpace ws;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (const int rc = check_entries(n, d_sequences, d_offsets)) return rc;
    if (n_tokens >= (size_t(1) << 31)) return fail(SVSX_INVALID_ARGUMENT, "too many rows in one call");
    if (n_tokens > 0 && !d_slots) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (n == 0 && n_tokens == 0) return SVSX_SUCCESS;
    if (const int rc = carve(a, n, d_workspace, workspace_bytes, &ws)) return rc;
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    // up to one row a thread the planner gives out the slots itself (64 sequences, with freeing them: 64 rows 12.6 us against 14.0 with a second launch, 1024 rows 13.2 against 14.3, 4096 rows 20.4 against 14.7)
    const bool near = n > 0 && n_tokens <= kPlanThreads;
    if (n > 0)
        hipLaunchKernelGGL(extend_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, d_sequences, d_offsets, static_cast<int>(n), static_cast<int>(n_tokens), ws,
                           near && n_tokens > 0 ? d_slots : nullptr);
    if (n_tokens > 0 && !near)
        hipLaunchKernelGGL(slots_kernel, dim3(static_cast<uint32_t>((n_tokens + 255) / 256)), dim3(256), 0, s, a, d_sequences, d_offsets, static_cast<int>(n), static_cast<int>(n_tokens),
                           ws.start, d_slots);
    return launched("cache extend");
}

int svsx_cache_copy_device(const svsx_cache_desc* desc, const int32_t* d_sources, const int32_t* d_targets, size_t n, int share, void* d_workspace, size_t workspace_bytes,
                           void* hip_stream) {
    CacheArgs a;
    PlanSpace ws;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (const int rc = check_entries(n, d_sources, d_targets)) return rc;
    if (n == 0) return SVSX_SUCCESS;
    if (const int rc = carve(a, n, d_workspace, workspace_bytes, &ws)) return rc;
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipLaunchKernelGGL(copy_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, d_sources, d_targets, static_cast<int>(n), share ? 1 : 0, ws);
    const size_t w = page_word(a);
    auto kernel = w >= 16 ? copy_pages_kernel<uint4> : w >= 4 ? copy_pages_kernel<uint32_t> : copy_pages_kernel<uint16_t>;
    hipLaunchKernelGGL(kernel, dim3(kMoveBlocks), dim3(256), 0, s, a, d_sources, d_targets, static_cast<int>(n), share ? 1 : 0, ws);
    return launched("cache copy");
}

int svsx_cache_free_device(const svsx_cache_desc* desc, const int32_t* d_sequences, size_t n, void* hip_stream) {
    CacheArgs a;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (const int rc = check_entries(n, d_sequences, d_sequences)) return rc;
    if (n == 0) return SVSX_SUCCESS;
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    hipLaunchKernelGGL(free_kernel, dim3(static_cast<uint32_t>(n)), dim3(256), 0, static_cast<hipStream_t>(hip_stream), a, d_sequences, static_cast<int>(n));
    return launched("cache free");
}

int svsx_cache_compact_device(const svsx_cache_desc* desc, int32_t* d_moved, void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    CacheArgs a;
    PlanSpace ws;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (!d_moved) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (const int rc = carve(a, 0, d_workspace, workspace_bytes, &ws)) return rc;
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, ws, d_moved);
    const size_t w = page_word(a);
    auto kernel = w >= 16 ? compact_pages_kernel<uint4> : w >= 4 ? compact_pages_kernel<uint32_t> : compact_pages_kernel<uint16_t>;
    hipLaunchKernelGGL(kernel, dim3(kMoveBlocks), dim3(256), 0, s, a, d_moved, ws);
    return launched("cache compact");
}

int svsx_cache_write_device(const svsx_cache_desc* desc, size_t layer, const int64_t* d_slots, size_t n_tokens, const void* d_keys, size_t key_token_stride,
                            size_t key_head_stride, const void* d_values, size_t value_token_stride, size_t value_head_stride, void* hip_stream) {
    CacheArgs a;
    if (const int rc = check_cache(desc, &a)) return rc;
    if (layer >= desc->n_layers) return fail(SVSX_INVALID_ARGUMENT, "layer %zu of a cache of %zu layers", layer, desc->n_layers);
    if (n_tokens >= (size_t(1) << 31)) return fail(SVSX_INVALID_ARGUMENT, "too many rows in one call");
    if (n_tokens == 0) return SVSX_SUCCESS;
    if (!d_slots || !d_keys) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if ((desc->value_dim != 0) != (d_values != nullptr)) return fail(SVSX_INVALID_ARGUMENT, "values are given exactly where the cache holds values");
    const size_t es = paged_dtype_size(desc->dtype), block = static_cast<size_t>(a.n_pages) * a.n_heads * a.page_size;
    WriteArgs w = {};
    w.slots = d_slots;
    w.src[0] = static_cast<const unsigned char*>(d_keys);
    w.src[1] = static_cast<const unsigned char*>(d_values);
    w.dst[0] = a.keys + layer * block * a.key_row_bytes;
    w.dst[1] = a.value_row_bytes ? a.values + layer * block * a.value_row_bytes : nullptr;
    w.token_bytes[0] = key_token_stride * es;
    w.token_bytes[1] = value_token_stride * es;
    w.head_bytes[0] = key_head_stride * es;
    w.head_bytes[1] = value_head_stride * es;
    const size_t word = word_of({reinterpret_cast<size_t>(d_keys), reinterpret_cast<size_t>(d_values), reinterpret_cast<size_t>(w.dst[0]), reinterpret_cast<size_t>(w.dst[1]),
                                 w.token_bytes[0], w.token_bytes[1], w.head_bytes[0], w.head_bytes[1], a.key_row_bytes, a.value_row_bytes});
    const size_t wide = word >= 16 ? 16 : word >= 4 ? 4 : 2;
    w.row_words[0] = static_cast<uint32_t>(a.key_row_bytes / wide);
    w.row_words[1] = static_cast<uint32_t>(a.value_row_bytes / wide);
    w.n_tokens = static_cast<uint32_t>(n_tokens);
    w.n_heads = a.n_heads;
    w.page_size = a.page_size;
    w.n_pages = a.n_pages;
    const size_t per_token = static_cast<size_t>(std::max(w.row_words[0], w.row_words[1])) * a.n_heads;
    if (per_token >= (size_t(1) << 31)) return fail(SVSX_INVALID_ARGUMENT, "a row of all heads has %zu words, 2^31 - 1 at most", per_token);
    const size_t blocks = std::min((n_tokens * per_token + 255) / 256, kWriteBlocks);
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    auto kernel = wide == 16 ? write_kernel<uint4> : wide == 4 ? write_kernel<uint32_t> : write_kernel<uint16_t>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks), d_values ? 2 : 1), dim3(256), 0, static_cast<hipStream_t>(hip_stream), w);
    return launched("cache write");
}

} // extern "C"
