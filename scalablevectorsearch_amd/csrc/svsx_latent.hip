// svsx_latent.hip -- latent attention in its expanded form, for prompts (include/svsx.h: svsx_latent_expanded_device).
//
// Two launches.  The first expands: keys K[head][row][dim] (the head's projection of the latent vector, then the rotary part, then zeros up to DK columns) and TRANSPOSED
// values V[head][column][row], products of 128 x 128 tiles; and it writes the list of query tiles, because only the device knows the sequences' offsets.  The second
// attends: prompts are long, so the products are large and the matrix units bound both.
#include "svsx_host.h"
#include "svsx_mfma.h"
#include <type_traits>

namespace svsx {
namespace {

struct ExpandedArgs {
    const void* queries;
    const void* rows;
    const void* w_key;
    const void* w_value;
    const int32_t* query_offsets;
    const int32_t* row_offsets;
    void* out;
    size_t query_stride, query_head_stride, row_stride;
    uint32_t n_sequences, n_tokens, n_rows, n_heads, nope, rope, rank, dv;
    float scale;
    int causal, keep_rest;
    int wide_queries, wide_out; // rows begin at 16-byte boundaries and are whole 16-byte words
};

// One query and head of a workgroup at a time, in the latent space: w_key applied to the query, w_value to the result.  For heads of more than 256 columns.
template <typename T> __device__ __forceinline__ void one_query(const ExpandedArgs& a, uint32_t h, uint32_t t, RowsShared& sm) {
    T* out = static_cast<T*>(a.out) + (static_cast<size_t>(t) * a.n_heads + h) * a.dv;
    int lo = 0, hi = static_cast<int>(a.n_sequences); // the last sequence whose queries begin at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.query_offsets[mid] <= static_cast<int32_t>(t)) lo = mid;
        else hi = mid;
    }
    const int32_t ti = static_cast<int32_t>(t);
    const bool mine = a.n_sequences > 0 && ti >= a.query_offsets[lo] && ti < a.query_offsets[lo + 1];
    if (!mine) {
        if (!a.keep_rest)
            for (uint32_t c = threadIdx.x; c < a.dv; c += 256) out[c] = from_f32<T>(0.0f);
        return;
    }
    const int32_t r0 = a.row_offsets[lo], r1 = a.row_offsets[lo + 1], last = r1 - (a.query_offsets[lo + 1] - ti); // its own row, in the array
    const int32_t end = a.causal ? last + 1 : r1;
    const T* q = static_cast<const T*>(a.queries) + t * a.query_stride + h * a.query_head_stride;
    const T* wk = static_cast<const T*>(a.w_key) + static_cast<size_t>(h) * a.nope * a.rank;
    const T* wv = static_cast<const T*>(a.w_value) + static_cast<size_t>(h) * a.dv * a.rank;
    for (uint32_t c = threadIdx.x; c < a.rank; c += 256) {
        float x = 0.0f;
        for (uint32_t d = 0; d < a.nope; ++d) x = fmaf(to_f32(q[d]), to_f32(wk[static_cast<size_t>(d) * a.rank + c]), x);
        sm.q[c] = x;
    }
    for (uint32_t c = threadIdx.x; c < a.rope; c += 256) sm.q[a.rank + c] = to_f32(q[a.nope + c]);
    __syncthreads();
    const T* rows = static_cast<const T*>(a.rows);
    const int32_t from = r0 < 0 ? 0 : r0, to = end < static_cast<int32_t>(a.n_rows) ? end : static_cast<int32_t>(a.n_rows);
    auto row_of = [&](uint32_t r) { return rows + static_cast<size_t>(from + r) * a.row_stride; };
    attend_rows<T>(sm, to > from ? static_cast<uint32_t>(to - from) : 0u, a.rank + a.rope, a.rank, a.scale, row_of, row_of);
    for (uint32_t c = threadIdx.x; c < a.dv; c += 256) {
        float x = 0.0f;
        for (uint32_t d = 0; d < a.rank; ++d) x = fmaf(sm.out[0][d], to_f32(wv[static_cast<size_t>(c) * a.rank + d]), x);
        out[c] = from_f32<T>(x);
    }
}

template <typename T> __global__ __launch_bounds__(256) void expanded_head_kernel(const ExpandedArgs a) {
    __shared__ RowsShared sm;
    for (uint32_t item = blockIdx.x; item < a.n_heads * a.n_tokens; item += gridDim.x) {
        one_query<T>(a, item % a.n_heads, item / a.n_heads, sm);
        __syncthreads(); // what the next query's threads write to has been read
    }
}

struct __align__(16) Tile { // of queries: all that the second launch needs to know of its sequence
    int32_t first, end;      // queries [first, end): the tile's first one, the sequence's last + 1
    int32_t begin, rows_end; // its rows, inside the array
    int32_t shift;           // query t's own row is t + shift
    int32_t unused[3];
};

struct Space { // the first launch's results
    void* keys;      // [head][key_rows][DK]
    void* values;    // [head][DV][value_rows]
    Tile* tiles;
    uint32_t* count;  // of tiles
    uint4* beyond;    // float16: per workgroup that multiplies (keys, then values) and wave of it, whether a finite result of its 128 x 128 is infinite in the row type
    size_t key_rows, value_rows; // at least n_rows + 64: a tile of rows may begin at the last one
    uint32_t dk, dv, most_tiles, tile_queries;
};

struct ExpandGrid { // workgroups of the first launch: keys, values, rotary parts, then one for the tiles
    uint32_t key_i, keys, value_i, values, copies;
};

// A plane in LDS is rows of 128 bytes (8 words of 16), in groups of eight rows that lie 16 bytes further apart than they are long; in the third and fourth
// row of four the two 64-byte halves are exchanged.  Eight lanes that read the same word of rows 0 .. 3 and 8 .. 11 (or 4 .. 7 and 12 .. 15: row32) meet in no bank, and a load
// straight from HBM fills a group in whole 64-byte pieces.
constexpr uint32_t kGroupBytes = 1024 + 16;
__device__ __forceinline__ uint32_t plane_at(uint32_t r, uint32_t word) { return (r >> 3) * kGroupBytes + (r & 7) * 128 + ((word ^ (r & 2) << 1) << 4); }
template <typename T> constexpr int kPlaneCols = 128 / sizeof(T);
template <typename T> constexpr int kSteps = kPlaneCols<T> / 16; // of product32 in a plane's columns

// the fragment of step `step` of row r of a plane for this half of the lanes
template <typename T> __device__ __forceinline__ Frag<T> plane_frag(const unsigned char* plane, uint32_t r, uint32_t step, uint32_t half) {
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const Frag<T>*>(plane + plane_at(r, step * 2 + half));
    } else {
        Frag<T> f;
        *reinterpret_cast<f32x4*>(&f) = *reinterpret_cast<const f32x4*>(plane + plane_at(r, step * 4 + half * 2));
        *(reinterpret_cast<f32x4*>(&f) + 1) = *reinterpret_cast<const f32x4*>(plane + plane_at(r, step * 4 + half * 2 + 1));
        return f;
    }
}

// 16 bytes of a row from column col on, zeros beyond dim
template <typename T> struct WordOf { typedef Frag<T> type; };
template <> struct WordOf<float> { typedef f32x4 type; };
template <typename T> using Word = typename WordOf<T>::type;
template <typename T, bool Wide> __device__ __forceinline__ Word<T> load_word(const T* row, uint32_t col, uint32_t dim) {
    constexpr uint32_t kElems = 16 / sizeof(T);
    Word<T> w = {};
    if constexpr (Wide) {
        if (col < dim) w = *reinterpret_cast<const Word<T>*>(row + col);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kElems; ++j)
            if (col + j < dim) w[j] = row[col + j];
    }
    return w;
}

// Highest bits (of each 16 for the 16-bit types) that are set where an element's exponent is all ones: one more at the exponent's lowest bit carries into the sign's place.
template <typename T> __device__ __forceinline__ uint32_t not_finite(const Frag<T>& f) {
    constexpr uint32_t kOne = sizeof(T) == 4 ? 0x00800000u : std::is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u, kSign = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    uint32_t word[sizeof(Frag<T>) / 4], bits = 0;
    __builtin_memcpy(word, &f, sizeof(f));
#pragma unroll
    for (uint32_t x : word) bits |= (x & ~kSign) + kOne;
    return bits & kSign;
}

// Float16 holds 65504 at most, and a projected row may be larger although its products with queries, or its weighted mean, are ordinary numbers.  (bfloat16 has float32's range.)
template <typename T> inline constexpr bool kNarrow = std::is_same<T, _Float16>::value;

// C[i][j] = sum_k A[i][k] B[j][k] for one 128 x 128 tile; four waves of 64 x 64.  row_a(i) / row_b(j): the row, NULL = zeros.  put(i, j, v): eight consecutive i of one j.
// Returns whether a finite sum of the wave's part is infinite in a row type of less range (false for the other types, without asking).
// The next 128 bytes of every row are on their way to registers while these are multiplied.  8190 rows of rank 512 for 32 heads (68.7 GFLOP): 114 us, 600 TFLOP/s, less than half of what a library product reaches; LDS is busy one and a
// half times as long as the matrix units.  Two buffers and one barrier a step were measured in place of one buffer: 333 tokens 25.4 -> 27.3 us then, as fewer workgroups fit a compute unit.
template <typename T, bool Wide, typename A, typename B, typename P> __device__ __forceinline__ bool product_tile(unsigned char* lds, uint32_t depth, A row_a, B row_b, P put) {
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5, r = row32(lane);
    unsigned char* const plane_a = lds;
    unsigned char* const plane_b = lds + 16 * kGroupBytes;
    const T* rows[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        rows[0][i] = row_a((t >> 3) + 32 * i);
        rows[1][i] = row_b((t >> 3) + 32 * i);
    }
    Word<T> next[2][4];
    auto fetch = [&](uint32_t col) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) next[s][i] = rows[s][i] ? load_word<T, Wide>(rows[s][i], col + (t & 7) * (16 / sizeof(T)), depth) : Word<T>{};
    };
    f32x16 c[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i >> 1][i & 1] = f32x16{};
    fetch(0);
    for (uint32_t col = 0; col < depth; col += kPlaneCols<T>) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *reinterpret_cast<Word<T>*>(plane_a + plane_at((t >> 3) + 32 * i, t & 7)) = next[0][i];
            *reinterpret_cast<Word<T>*>(plane_b + plane_at((t >> 3) + 32 * i, t & 7)) = next[1][i];
        }
        __syncthreads();
        if (col + kPlaneCols<T> < depth) fetch(col + kPlaneCols<T>);
#pragma unroll
        for (int s = 0; s < kSteps<T>; ++s) {
            Frag<T> fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = plane_frag<T>(plane_a, (wave & 1) * 64 + i * 32 + r, s, half);
                fb[i] = plane_frag<T>(plane_b, (wave >> 1) * 64 + i * 32 + r, s, half);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i >> 1][i & 1] = product32(fa[i >> 1], fb[i & 1], c[i >> 1][i & 1]);
        }
    }
    bool beyond = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                Frag<T> v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = from_f32<T>(c[i][j][8 * k + e]);
                if (kNarrow<T> && not_finite<T>(v)) // 65520, halfway to 2^16, is the first that is rounded up
#pragma unroll
                    for (int e = 0; e < 8; ++e) beyond |= fabsf(c[i][j][8 * k + e]) >= 65520.0f && fabsf(c[i][j][8 * k + e]) < INFINITY;
                put((wave & 1) * 64 + i * 32 + 16 * k + 8 * half, (wave >> 1) * 64 + j * 32 + r, v);
            }
    return kNarrow<T> && __any(beyond);
}

// the queries of sequence i, inside the array
__device__ __forceinline__ void queries_of(const ExpandedArgs& a, uint32_t i, uint32_t* begin, uint32_t* end) {
    const int32_t b = a.query_offsets[i], e = a.query_offsets[i + 1], n = static_cast<int32_t>(a.n_tokens);
    *begin = static_cast<uint32_t>(b < 0 ? 0 : b < n ? b : n);
    *end = static_cast<uint32_t>(e < static_cast<int32_t>(*begin) ? static_cast<int32_t>(*begin) : e < n ? e : n);
}

// the query tiles, sequence by sequence, and zeros for the queries of no sequence
template <typename T> __device__ __forceinline__ void list_tiles(const ExpandedArgs& a, const Space& w, uint32_t* sh) {
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t base = 0;
    for (uint32_t first = 0; first < a.n_sequences; first += 256) {
        uint32_t b = 0, e = 0;
        if (first + t < a.n_sequences) queries_of(a, first + t, &b, &e);
        const uint32_t n = (e - b + w.tile_queries - 1) / w.tile_queries;
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
        for (uint32_t k = 0; k < 4; ++k) {
            at += k < wave ? sh[k] : 0;
            base += sh[k];
        }
        if (n > 0) {
            const int32_t rb = a.row_offsets[first + t], re = a.row_offsets[first + t + 1], n_rows = static_cast<int32_t>(a.n_rows);
            Tile tile = {0, static_cast<int32_t>(e), rb < 0 ? 0 : rb, re < n_rows ? re : n_rows, re - a.query_offsets[first + t + 1], {}};
            for (uint32_t k = 0; k < n; ++k) {
                tile.first = static_cast<int32_t>(b + k * w.tile_queries);
                if (at + k < w.most_tiles) w.tiles[at + k] = tile;
            }
        }
    }
    if (t == 0) *w.count = base < w.most_tiles ? base : w.most_tiles;
}

template <typename T, bool Wide> __global__ __launch_bounds__(256) void expand_kernel(const ExpandedArgs a, const Space w, const ExpandGrid grid) {
    __shared__ __align__(16) unsigned char lds[2 * 16 * kGroupBytes];
    uint32_t block = blockIdx.x;
    const T* rows = static_cast<const T*>(a.rows);
    T* keys = static_cast<T*>(w.keys);
    T* values = static_cast<T*>(w.values);
    auto row_of = [&](uint32_t r) -> const T* { // NULL, zeros, for rows of no sequence, which may hold anything
        const int32_t begin = a.n_sequences ? a.row_offsets[0] : 0, end = a.n_sequences ? a.row_offsets[a.n_sequences] : 0;
        return r < a.n_rows && static_cast<int32_t>(r) >= begin && static_cast<int32_t>(r) < end ? rows + static_cast<size_t>(r) * a.row_stride : nullptr;
    };
    if (block < grid.keys) { // i: (head, column), j: row
        const uint32_t i0 = block % grid.key_i * 128, j0 = block / grid.key_i * 128, n = a.n_heads * a.nope;
        const T* wk = static_cast<const T*>(a.w_key);
        const bool beyond = product_tile<T, Wide>(
            lds, a.rank, [&](uint32_t i) { return i0 + i < n ? wk + static_cast<size_t>(i0 + i) * a.rank : nullptr; },
            [&](uint32_t j) { return row_of(j0 + j); },
            [&](uint32_t i, uint32_t j, const Frag<T>& v) {
                if (j0 + j >= a.n_rows) return;
                if (a.nope % 8 == 0) {
                    const uint32_t h = (i0 + i) / a.nope, col = (i0 + i) % a.nope;
                    if (h < a.n_heads) *reinterpret_cast<Frag<T>*>(keys + (h * w.key_rows + j0 + j) * w.dk + col) = v;
                } else {
                    for (uint32_t e = 0; e < 8; ++e) {
                        const uint32_t h = (i0 + i + e) / a.nope, col = (i0 + i + e) % a.nope;
                        if (h < a.n_heads) keys[(h * w.key_rows + j0 + j) * w.dk + col] = v[e];
                    }
                }
            });
        if (kNarrow<T> && (threadIdx.x & 63) == 0) reinterpret_cast<uint32_t*>(w.beyond + blockIdx.x)[threadIdx.x >> 6] = beyond;
        return;
    }
    block -= grid.keys;
    if (block < grid.values) { // i: row, j: (head, column); zeros in columns beyond the head's and rows beyond the last
        const uint32_t i0 = block % grid.value_i * 128, j0 = block / grid.value_i * 128, n = a.n_heads * w.dv;
        const T* wv = static_cast<const T*>(a.w_value);
        const bool beyond = product_tile<T, Wide>(
            lds, a.rank, [&](uint32_t i) { return row_of(i0 + i); },
            [&](uint32_t j) {
                const uint32_t h = (j0 + j) / w.dv, col = (j0 + j) % w.dv;
                return j0 + j < n && col < a.dv ? wv + (static_cast<size_t>(h) * a.dv + col) * a.rank : nullptr;
            },
            [&](uint32_t i, uint32_t j, const Frag<T>& v) {
                if (i0 + i < w.value_rows && j0 + j < n) *reinterpret_cast<Frag<T>*>(values + static_cast<size_t>(j0 + j) * w.value_rows + i0 + i) = v;
            });
        if (kNarrow<T> && (threadIdx.x & 63) == 0) reinterpret_cast<uint32_t*>(w.beyond + blockIdx.x)[threadIdx.x >> 6] = beyond;
        return;
    }
    block -= grid.values;
    if (block < grid.copies) { // the rotary part behind every head's columns, zeros behind that
        constexpr uint32_t kElems = 16 / sizeof(T);
        const bool words = Wide && a.nope % kElems == 0 && a.rope % kElems == 0;
        const uint32_t step = words ? kElems : 1, per_row = (w.dk - a.nope) / step;
        const uint64_t all = static_cast<uint64_t>(a.n_heads) * a.n_rows * per_row;
        for (uint64_t at = static_cast<uint64_t>(block) * 256 + threadIdx.x; at < all; at += static_cast<uint64_t>(grid.copies) * 256) {
            const uint32_t col = static_cast<uint32_t>(at % per_row) * step;
            const uint64_t hr = at / per_row;
            const uint32_t r = static_cast<uint32_t>(hr % a.n_rows), h = static_cast<uint32_t>(hr / a.n_rows);
            const T* from = rows + static_cast<size_t>(r) * a.row_stride + a.rank + col;
            T* to = keys + (h * w.key_rows + r) * w.dk + a.nope + col;
            if (words) *reinterpret_cast<Word<T>*>(to) = col < a.rope ? *reinterpret_cast<const Word<T>*>(from) : Word<T>{};
            else *to = col < a.rope ? *from : from_f32<T>(0.0f);
        }
        if (!a.keep_rest) { // queries before the first sequence and behind the last
            uint32_t b = a.n_tokens, e = a.n_tokens, unused;
            if (a.n_sequences > 0) {
                queries_of(a, 0, &b, &unused);
                queries_of(a, a.n_sequences - 1, &unused, &e);
                e = e < b ? b : e;
            }
            const size_t per_query = static_cast<size_t>(a.n_heads) * a.dv, rest = (b + (a.n_tokens - e)) * per_query;
            T* out = static_cast<T*>(a.out);
            for (size_t at = static_cast<size_t>(block) * 256 + threadIdx.x; at < rest; at += static_cast<size_t>(grid.copies) * 256)
                out[at < b * per_query ? at : at + (e - b) * per_query] = from_f32<T>(0.0f);
        }
        return;
    }
    list_tiles<T>(a, w, reinterpret_cast<uint32_t*>(lds));
}

// One workgroup: NW waves of 32 queries of one head, over the rows they see in tiles of 64 (float32: 32).
//   S^T = K Q^T    rows x queries, queries as fragments in registers; with row32, a lane's results are eight consecutive rows at a time for its query:
//   O^T = V^T P^T  the probabilities are the next product's fragments where they are.
// A query is a lane's column throughout, so its maximum, sum and rescaling need one exchange between two lanes.  Per 64 rows a wave has 1280 cycles of products
// (DK 192, DV 128) against 320 of LDS reads, which eight waves share, and about 1000 of softmax on the vector units: so of the two waves on a SIMD, one does its products (a tile's
// scores and the last tile's values) while the other does its softmax, and they change over at a barrier.
// 4095 queries on 8190 rows, 32 heads, bfloat16: 433 us, 1.19 PFLOP/s, 87 % of what an 8192^3 library product reaches.  The call: 547 us; float16 574; float32 4.74 ms, 123 TFLOP/s; bfloat16 with 128 heads
// 2.36 ms.  (192, 128) with eight waves spills 1 to 3 registers at its start, no other variant any.
template <typename T, int DK, int DV, int NW> struct PromptLayout {
    static constexpr uint32_t kRows = kPlaneCols<T>; // of a tile: a plane of V^T
    static constexpr int kKeyPlanes = DK / kPlaneCols<T>, kTiles = kRows / 32;
    static constexpr uint32_t kGroups = kRows / 8, kKeyPlane = kGroups * kGroupBytes, kKeyBytes = kKeyPlanes * kKeyPlane, kValueBytes = DV / 8 * kGroupBytes;
    static constexpr uint32_t kAhead = 3 * kKeyBytes + 2 * kValueBytes <= 160 * 1024 ? 2 : 1; // tiles that keys are brought in ahead of their use
    static constexpr uint32_t kBytes = (kAhead + 1) * kKeyBytes + 2 * kValueBytes;
    static_assert(kBytes <= 160 * 1024 && kGroups % 4 == 0 && DV % 32 == 0, "LDS; loads of four waves");
    static_assert(!kNarrow<T> || kBytes >= NW * 2 * kMaxDim * sizeof(float), "latent_query's LDS");
};
// One query by one wave, over the expanded rows [begin, last] alone: its lanes across the columns.  Slow: a NaN in one row of 8190 that only the last of 4095 queries sees takes the call from 0.6 to 157 ms.
template <typename T, int DK, int DV> __device__ void slow_query(const ExpandedArgs& a, const Space& w, uint32_t t, uint32_t h, int32_t begin, int32_t last) {
    const uint32_t lane = threadIdx.x & 63, dk = a.nope + a.rope;
    const T* row = static_cast<const T*>(a.queries) + t * a.query_stride + h * a.query_head_stride;
    const T* keys = static_cast<const T*>(w.keys) + h * w.key_rows * DK;
    const T* values = static_cast<const T*>(w.values) + static_cast<size_t>(h) * DV * w.value_rows;
    float q[DK / 64], o[DV / 64], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < DK / 64; ++i) q[i] = lane + 64 * i < dk ? to_f32(row[lane + 64 * i]) : 0.0f;
#pragma unroll
    for (int i = 0; i < DV / 64; ++i) o[i] = 0.0f;
    for (int32_t r = begin; r <= last; ++r) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < DK / 64; ++i) s = fmaf(q[i], to_f32(keys[static_cast<size_t>(r) * DK + lane + 64 * i]), s);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
        s *= a.scale;
        if (s == -INFINITY) continue;
        const float raised = s > top || s != s ? s : top, was = expf(top - raised), p = expf(s - raised);
        top = raised;
        sum = fmaf(sum, was, p);
#pragma unroll
        for (int i = 0; i < DV / 64; ++i) o[i] = fmaf(p, to_f32(values[(lane + 64 * i) * w.value_rows + r]), o[i] * was);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out) + (static_cast<size_t>(t) * a.n_heads + h) * a.dv;
#pragma unroll
    for (int i = 0; i < DV / 64; ++i)
        if (lane + 64 * i < a.dv) out[lane + 64 * i] = from_f32<T>(o[i] * inv);
}

// Whether an expanded key or value of head h, in rows begin .. last, is infinite only for the row type's range (with what shares its workgroup in the first launch).  Every
// wave asks for itself, and gets the same answer.  Asking, beside the first rows' loads, takes 333 tokens of 16 heads from 26.4 to 27.5 us; 4095 on 8190 rows, 32 heads, are as they were.
__device__ __forceinline__ bool any_beyond(const ExpandedArgs& a, const Space& w, const ExpandGrid& grid, uint32_t h, int32_t begin, int32_t last) {
    bool beyond = false;
    if (begin <= last) {
        const uint32_t r0 = static_cast<uint32_t>(begin) / 128, rows = static_cast<uint32_t>(last) / 128 - r0 + 1;
        const uint32_t k0 = h * a.nope / 128, ks = a.nope ? ((h + 1) * a.nope - 1) / 128 - k0 + 1 : 0; // workgroups across the head's columns
        const uint32_t v0 = h * w.dv / 128, vs = ((h + 1) * w.dv - 1) / 128 - v0 + 1;
        auto at = [&](uint32_t block) {
            const uint4 x = w.beyond[block];
            beyond |= (x.x | x.y | x.z | x.w) != 0;
        };
        for (uint32_t r = threadIdx.x & 63; r < rows; r += 64) {
            for (uint32_t k = 0; k < ks; ++k) at((r0 + r) * grid.key_i + k0 + k);
            for (uint32_t v = 0; v < vs; ++v) at(grid.keys + (v0 + v) * grid.value_i + r0 + r);
        }
    }
    return __any(beyond);
}

// The softmax of one wave's query over rows [begin, last] in the latent space: the query `q` and the weighted sum of rows `o` are in LDS, 8 columns a lane and 512 a chunk; four rows at a time.
template <typename T, bool Wide> __device__ __forceinline__ void latent_rows(const ExpandedArgs& a, int32_t begin, int32_t last, const float* q, float* o, float* total) {
    constexpr int kBatch = 4, kChunks = kMaxDim / 512;
    const uint32_t lane = threadIdx.x & 63, width = a.rank + a.rope;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 1
    for (int32_t r = begin; r <= last; r += kBatch) {
        Frag<T> x[kBatch][kChunks];
        float s[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const T* row = static_cast<const T*>(a.rows) + static_cast<size_t>(min(r + b, last)) * a.row_stride;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) x[b][c] = load_frag<T, Wide>(row, c * 512 + lane * 8, width);
            s[b] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const f32x8 mine = *reinterpret_cast<const f32x8*>(q + c * 512 + lane * 8);
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[b] = fmaf(mine[e], to_f32(x[b][c][e]), s[b]);
        }
        float raised = top;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) s[b] += __shfl_xor(s[b], off);
            s[b] = r + b <= last ? s[b] * a.scale : -INFINITY;
            raised = s[b] > raised || s[b] != s[b] ? s[b] : raised;
        }
        if (raised == -INFINITY) continue; // no weight yet
        const float was = top == -INFINITY ? 0.0f : expf(top - raised);
        top = raised;
        sum *= was;
        f32x8 mine[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) mine[c] = *reinterpret_cast<const f32x8*>(o + c * 512 + lane * 8) * was;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (s[b] == -INFINITY) continue; // no weight; it must not become the difference of two infinities
            const float p = expf(s[b] - top);
            sum += p;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) mine[c][e] = fmaf(p, to_f32(x[b][c][e]), mine[c][e]);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) *reinterpret_cast<f32x8*>(o + c * 512 + lane * 8) = mine[c];
    }
    *total = sum;
}

// One query by one wave in the latent space, where nothing is rounded on the way: w_key applied to the query, rows [begin, last], w_value to the result.  The query and the sums are in the
// wave's own `lds` (2 kMaxDim floats), so that this rare path takes no registers from the usual one.  One row of 8190 whose keys are too large, 4095 queries, 32 heads: 121 ms where the last 126 queries see
// its 128 rows, 192 ms where 2190 do (a row at a time, a column a lane: 959 and 1438 ms; the usual way 0.57).
template <typename T> __device__ __forceinline__ void latent_query(const ExpandedArgs& a, uint32_t t, uint32_t h, int32_t begin, int32_t last, float* lds) {
    const uint32_t lane = threadIdx.x & 63, width = a.rank + a.rope;
    const T* query = static_cast<const T*>(a.queries) + t * a.query_stride + h * a.query_head_stride;
    float *const q = lds, *const o = lds + kMaxDim;
#pragma unroll 1
    for (uint32_t c = lane; c < kMaxDim; c += 64) {
        const T* w = static_cast<const T*>(a.w_key) + static_cast<size_t>(h) * a.nope * a.rank + c;
        float x = c >= a.rank && c < width ? to_f32(query[a.nope + c - a.rank]) : 0.0f;
        if (c < a.rank)
#pragma unroll 8
            for (uint32_t d = 0; d < a.nope; ++d) x = fmaf(to_f32(query[d]), to_f32(w[static_cast<size_t>(d) * a.rank]), x);
        q[c] = x;
        o[c] = 0.0f;
    }
    __threadfence_block(); // a lane reads what others wrote
    float sum;
    if (width % 8 == 0 && ((reinterpret_cast<size_t>(a.rows) | a.row_stride * sizeof(T)) & 15) == 0) latent_rows<T, true>(a, begin, last, q, o, &sum);
    else latent_rows<T, false>(a, begin, last, q, o, &sum);
    __threadfence_block();
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
    for (uint32_t c = lane; c < a.dv; c += 64) {
        const T* w = static_cast<const T*>(a.w_value) + (static_cast<size_t>(h) * a.dv + c) * a.rank;
        float y = 0.0f;
#pragma unroll 8
        for (uint32_t d = 0; d < a.rank; ++d) y = fmaf(o[d], to_f32(w[d]), y);
        static_cast<T*>(a.out)[(static_cast<size_t>(t) * a.n_heads + h) * a.dv + c] = from_f32<T>(y * inv);
    }
    __threadfence_block(); // the next query's sums go where these were
}

template <typename T, int DK, int DV, int NW> __global__ __launch_bounds__(NW * 64) void prompt_kernel(const ExpandedArgs a, const Space w, const ExpandGrid grid) {
    typedef PromptLayout<T, DK, DV, NW> L;
    extern __shared__ __align__(16) unsigned char lds[];
    const uint32_t count = *w.count, turn = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads; // a head's tiles on one of the eight L2s where heads are a multiple of 8
    if (turn >= count) return;
    const Tile tile = w.tiles[count - 1 - turn]; // a sequence's last queries see the most rows: they go first
    const uint32_t q0 = __builtin_amdgcn_readfirstlane(tile.first), qe = __builtin_amdgcn_readfirstlane(tile.end);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r = row32(lane);
    const int32_t begin = __builtin_amdgcn_readfirstlane(tile.begin), end = __builtin_amdgcn_readfirstlane(tile.rows_end), shift = __builtin_amdgcn_readfirstlane(tile.shift);
    auto sees = [&](uint32_t t) { // the last row that query t sees; less than begin: none
        const int32_t own = static_cast<int32_t>(t) + shift;
        return a.causal && own < end - 1 ? own : end - 1;
    };
    const uint32_t q_last = min(qe, q0 + NW * 32) - 1, mine = min(q0 + wave * 32 + (lane & 31), q_last);
    const int32_t see = sees(mine);
    const int32_t wave_first = __builtin_amdgcn_readfirstlane(sees(min(q0 + wave * 32, q_last))), wave_last = __builtin_amdgcn_readfirstlane(sees(min(q0 + wave * 32 + 31, q_last)));
    const int32_t base0 = begin & ~7, group_last = __builtin_amdgcn_readfirstlane(sees(q_last)); // V^T is read in 16-byte words

    Frag<T> q[DK / 16];
    {
        const T* row = static_cast<const T*>(a.queries) + mine * a.query_stride + h * a.query_head_stride;
        const uint32_t dk = a.nope + a.rope;
#pragma unroll
        for (int s = 0; s < DK / 16; ++s) {
            q[s] = a.wide_queries ? load_frag<T, true>(row, s * 16 + half * 8, dk) : load_frag<T, false>(row, s * 16 + half * 8, dk);
            // the scale's sign goes into the queries (exactly), so that the largest product has the largest score; so does a scale of zero
            if (!(a.scale > 0.0f)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) q[s][e] = a.scale < 0.0f ? -q[s][e] : from_f32<T>(0.0f);
            }
        }
    }
    // the compiler is to wait for the queries here: in the loop, where it cannot tell them from the rows on their way, it would wait for both
#pragma unroll
    for (int s = 0; s < DK / 16; ++s) asm volatile("" : "+v"(q[s]));
    f32x16 o[DV / 32];
#pragma unroll
    for (int d = 0; d < DV / 32; ++d) o[d] = f32x16{};
    float top = -INFINITY, sum = 0.0f;
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;

    const T* keys = static_cast<const T*>(w.keys) + h * w.key_rows * DK;
    const T* values = static_cast<const T*>(w.values) + static_cast<size_t>(h) * DV * w.value_rows;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_byte*)lds));
    // a lane's place in a group of eight rows: row lane / 8, and the word that belongs at lane % 8 there
    const uint32_t in_row = ((lane & 7) ^ (lane >> 3 & 2) << 1) * 16;
    const uint32_t key_offset = (lane >> 3) * (DK * sizeof(T)) + in_row, value_offset = (lane >> 3) * static_cast<uint32_t>(w.value_rows * sizeof(T)) + in_row;
    // Four waves bring in a tile's keys, or its values, 1 KB a load.  Issuing a load takes a wave about a hundred cycles, so it is done beside the softmax.
    const uint32_t of_four = wave & 3;
    unsigned char* const value_buffers = lds + (L::kAhead + 1) * L::kKeyBytes;
    auto bring_keys = [&](uint32_t buffer, int32_t base) {
        const T* from = keys + (static_cast<size_t>(base) + of_four * 8) * DK;
        const uint32_t to = lds0 + buffer * L::kKeyBytes + of_four * kGroupBytes;
#pragma unroll
        for (uint32_t k = 0; k < L::kKeyPlanes * L::kGroups; k += 4)
            direct_load(from + (k % L::kGroups) * 8 * DK + k / L::kGroups * kPlaneCols<T>, key_offset,
                        __builtin_amdgcn_readfirstlane(to + k / L::kGroups * L::kKeyPlane + k % L::kGroups * kGroupBytes));
    };
    auto bring_values = [&](uint32_t buffer, int32_t base) {
        const T* from = values + static_cast<size_t>(of_four) * 8 * w.value_rows + base;
        const uint32_t to = lds0 + (L::kAhead + 1) * L::kKeyBytes + buffer * L::kValueBytes + of_four * kGroupBytes;
#pragma unroll
        for (uint32_t k = 0; k < DV / 8; k += 4) direct_load(from + k * 8 * w.value_rows, value_offset, __builtin_amdgcn_readfirstlane(to + k * kGroupBytes));
    };

    // Where eight waves run, the second four are half a tile behind the first: tile i's products ("M": its scores, and tile i - 1's values) stand beside the other four's softmax
    // ("S") of i - 1 or i.  During its S(i) the first four bring in the keys of tile i + kAhead, the second four (or the only ones) the values of i + 1: the buffers
    // those go to were last read in M(i - 1) and M(i), which a barrier has ended for all.
    const bool paired = NW > 4, second = wave >= 4;
    const int32_t step = L::kRows;
    uint32_t key_buffer = 0, value_buffer = 0; // of this tile
    bool odd = false, pending = false, pending_edge = false; // a tile whose probabilities wait for its values
    f32x16 s[L::kTiles];
    Frag<T> p[2 * L::kTiles];
    auto add_values = [&](uint32_t buffer) {
        const unsigned char* vt = value_buffers + buffer * L::kValueBytes;
        if (pending_edge) { // values of rows that some query does not see: a weight of zero does not take away what is infinite or not a number
            uint32_t bits = 0;
#pragma unroll
            for (int d = 0; d < DV / 32; ++d)
#pragma unroll
                for (int k = 0; k < 2 * L::kTiles; ++k) bits |= not_finite<T>(plane_frag<T>(vt, d * 32 + r, k, half));
            odd |= __any(bits != 0);
        }
#pragma unroll
        for (int k = 0; k < 2 * L::kTiles; ++k)
#pragma unroll
            for (int d = 0; d < DV / 32; ++d) o[d] = product32(plane_frag<T>(vt, d * 32 + r, k, half), p[k], o[d]);
        reads_ahead<T, 2 * L::kTiles * (DV / 32), 4>();
    };
    if (base0 <= group_last) {
        if (!second) {
            bring_keys(0, base0);
            if (L::kAhead > 1 && base0 + step <= group_last) bring_keys(1, base0 + step);
            bring_values(0, base0);
        }
        if constexpr (kNarrow<T>) { // asked while the first rows are on their way
            if (any_beyond(a, w, grid, h, begin, group_last)) {
                direct_wait();
                __syncthreads();
                for (uint32_t t = q0 + wave * 32; t <= min(q_last, q0 + wave * 32 + 31); ++t) latent_query<T>(a, t, h, begin, sees(t), reinterpret_cast<float*>(lds) + wave * (2 * kMaxDim));
                return;
            }
        }
        direct_wait();
        lds_barrier();
        if (second) lds_barrier();
        for (int32_t base = base0; base <= group_last; base += step) {
            const bool active = base <= wave_last, edge = base < begin || base + step - 1 > wave_first;
            if (active) {
                const unsigned char* kt = lds + key_buffer * L::kKeyBytes;
#pragma unroll
                for (int x = 0; x < L::kTiles; ++x) s[x] = f32x16{};
#pragma unroll
                for (int k = 0; k < DK / 16; ++k)
#pragma unroll
                    for (int x = 0; x < L::kTiles; ++x) s[x] = product32(plane_frag<T>(kt + k / kSteps<T> * L::kKeyPlane, x * 32 + r, k % kSteps<T>, half), q[k], s[x]);
                reads_ahead<T, DK / 16 * L::kTiles, 4>();
            }
            if (pending) add_values(value_buffer ^ 1);
            if (second) direct_wait(); // the values of this tile, which M(i + 1) of the first four is about to read
            lds_barrier();
            if (!second) {
                if (L::kAhead > 1) direct_wait(); // what S(i - 1) brought: the keys of tile i + 1
                const int32_t far = base + static_cast<int32_t>(L::kAhead) * step;
                if (far <= group_last) bring_keys(key_buffer ? key_buffer - 1 : L::kAhead, far);
            }
            if ((!paired || second) && base + step <= group_last) bring_values(value_buffer ^ 1, base + step);
            if (active) {
                // register 8 i + e of s[x]: row base + 32 x + 16 i + 8 half + e
                if (edge) {
#pragma unroll
                    for (int x = 0; x < L::kTiles; ++x)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int32_t row = base + 32 * x + 16 * (i >> 3) + 8 * static_cast<int32_t>(half) + (i & 7);
                            if (row < begin || row > see) s[x][i] = -INFINITY;
                        }
                }
                float most = -INFINITY;
#pragma unroll
                for (int x = 0; x < L::kTiles; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, s[x][i]);
                most = fmaxf(most, __shfl_xor(most, 32)) * scale;
                if (__any(most > top + kSlack)) {
                    const float raised = fmaxf(top, most), shrink = top == -INFINITY ? 0.0f : exp2_fast(top - raised);
                    top = raised;
                    sum *= shrink;
#pragma unroll
                    for (int d = 0; d < DV / 32; ++d) o[d] *= shrink;
                }
                const float from = (top == -INFINITY ? 0.0f : top) - kLift<T>;
#pragma unroll
                for (int x = 0; x < L::kTiles; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float e = exp2_fast(fmaf(s[x][i], scale, -from));
                        sum += e;
                        p[2 * x + (i >> 3)][i & 7] = from_f32<T>(e);
                    }
            }
            pending = active;
            pending_edge = edge;
            if (!second && L::kAhead == 1) direct_wait();
            lds_barrier();
            key_buffer = key_buffer == L::kAhead ? 0 : key_buffer + 1;
            value_buffer ^= 1;
        }
        if (pending) add_values(value_buffer ^ 1);
        if (paired && !second) lds_barrier();
    }
    if (odd) { // anew, row by row, from the rows that each query sees
        for (uint32_t t = q0 + wave * 32; t <= min(q_last, q0 + wave * 32 + 31); ++t) slow_query<T, DK, DV>(a, w, t, h, begin, sees(t));
        return;
    }
    sum += __shfl_xor(sum, 32);
    if (q0 + wave * 32 + (lane & 31) > q_last) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(a.out) + (static_cast<size_t>(mine) * a.n_heads + h) * a.dv;
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t col = d * 32 + 16 * i + 8 * half;
            Frag<T> f;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = from_f32<T>(o[d][8 * i + e] * inv);
            if (a.wide_out) {
                if (col < a.dv) *reinterpret_cast<Frag<T>*>(out + col) = f;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    if (col + e < a.dv) out[col + e] = f[e];
            }
        }
}

int check_expanded(const svsx_expanded_desc* d, ExpandedArgs* a) {
    if (!d) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (d->struct_size != sizeof(svsx_expanded_desc))
        return fail(SVSX_INVALID_ARGUMENT, "svsx_expanded_desc.struct_size is %zu, expected %zu", d->struct_size, sizeof(svsx_expanded_desc));
    if (paged_dtype_size(d->dtype) == 0) return fail(SVSX_INVALID_ARGUMENT, "unsupported row dtype %d (float32, float16, bfloat16)", d->dtype);
    if (d->n_heads == 0 || d->n_heads > 65535) return fail(SVSX_INVALID_ARGUMENT, "n_heads must be in [1, 65535]");
    if (d->rank == 0 || d->value_dim == 0 || d->value_dim > kMaxDim || d->rank > kMaxDim || d->rope_dim > kMaxDim || d->rank + d->rope_dim > kMaxDim || d->nope_dim > kMaxDim ||
        d->nope_dim + d->rope_dim > kMaxDim || d->nope_dim + d->rope_dim == 0)
        return fail(SVSX_INVALID_ARGUMENT, "rank (%zu) + rope_dim (%zu), nope_dim (%zu) + rope_dim and value_dim (%zu) must be in [1, %d]", d->rank, d->rope_dim, d->nope_dim,
                    d->value_dim, kMaxDim);
    // grids have fewer than 2^32 threads: with these limits, and rows that fit the machine's memory once they are expanded, all of them do
    if (d->n_rows >= (size_t(1) << 27) - 128 || d->n_tokens >= size_t(1) << 29 || d->n_tokens * d->n_heads >= size_t(1) << 29 || d->n_sequences >= size_t(1) << 22 ||
        d->n_sequences * d->n_heads >= size_t(1) << 22)
        return fail(SVSX_INVALID_ARGUMENT, "too many queries, rows or sequences in one call (n_rows %zu, n_tokens %zu, n_sequences %zu, n_heads %zu)", d->n_rows, d->n_tokens, d->n_sequences, d->n_heads);
    if (!std::isfinite(d->scale)) return fail(SVSX_INVALID_ARGUMENT, "scale must be finite");
    if (d->n_tokens > 0 && (!d->d_queries || !d->d_out || !d->d_w_value || (d->nope_dim > 0 && !d->d_w_key))) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (d->n_tokens > 0 && d->n_sequences > 0 && (!d->d_query_offsets || !d->d_row_offsets || (d->n_rows > 0 && !d->d_rows))) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *a = ExpandedArgs{d->d_queries, d->d_rows, d->d_w_key, d->d_w_value, d->d_query_offsets, d->d_row_offsets, d->d_out, d->query_stride, d->query_head_stride, d->row_stride,
                      static_cast<uint32_t>(d->n_sequences), static_cast<uint32_t>(d->n_tokens), static_cast<uint32_t>(d->n_rows), static_cast<uint32_t>(d->n_heads),
                      static_cast<uint32_t>(d->nope_dim), static_cast<uint32_t>(d->rope_dim), static_cast<uint32_t>(d->rank), static_cast<uint32_t>(d->value_dim), d->scale,
                      d->causal, d->keep_rest, 0, 0};
    const size_t es = paged_dtype_size(d->dtype), dk = d->nope_dim + d->rope_dim;
    a->wide_queries = dk % 8 == 0 && ((reinterpret_cast<size_t>(d->d_queries) | d->query_stride * es | d->query_head_stride * es) & 15) == 0;
    a->wide_out = d->value_dim % 8 == 0 && (reinterpret_cast<size_t>(d->d_out) & 15) == 0;
    return SVSX_SUCCESS;
}

// How a call is answered; decided from sizes, types, strides and addresses alone.
struct PromptRoute {
    bool tiles; // on the matrix units; else one workgroup per query and head (heads of more than 256 columns)
    bool wide;
    int dk, dv, waves;
    Space space;
    ExpandGrid grid;
    size_t values_at, tiles_at, count_at, beyond_at, bytes;
};

PromptRoute route_of(const ExpandedArgs& a, int dtype) {
    PromptRoute r = {};
    const size_t es = paged_dtype_size(dtype);
    const uint32_t dk = a.nope + a.rope;
    r.tiles = dk <= 256 && a.dv <= 256;
    if (!r.tiles) return r;
    r.dk = dk <= 128 && a.dv <= 128 ? 128 : dk <= 192 && a.dv <= 128 ? 192 : 256;
    r.dv = r.dk == 256 ? 256 : a.dv <= 64 ? 64 : 128;
    const size_t elems = 16 / es;
    r.wide = a.rank % elems == 0 && ((reinterpret_cast<size_t>(a.rows) | reinterpret_cast<size_t>(a.w_key) | reinterpret_cast<size_t>(a.w_value) | a.row_stride * es) & 15) == 0;
    // Eight waves share a tile's rows where that leaves every compute unit a workgroup (causal prompts, 4 and 8 waves: 512 tokens, 16 heads 34 and 38 us; 1000, 32 heads 60 and 60; 2048, 32 heads
    // 125 and 115; 4096, 32 heads 325 and 243); float32 and 256-column heads have no registers for two waves a SIMD.
    r.waves = es == 2 && r.dk <= 192 && static_cast<uint64_t>(a.n_tokens) * a.n_heads >= 256 * 256 ? 8 : 4;
    Space& w = r.space;
    w.dk = r.dk;
    w.dv = r.dv;
    w.tile_queries = r.waves * 32;
    w.most_tiles = (a.n_tokens + w.tile_queries - 1) / w.tile_queries + a.n_sequences;
    w.key_rows = static_cast<size_t>(a.n_rows) + 64;
    w.value_rows = (static_cast<size_t>(a.n_rows) + 63) / 64 * 64 + 64;
    r.values_at = a.n_heads * w.key_rows * r.dk * es;
    r.tiles_at = r.values_at + a.n_heads * w.value_rows * r.dv * es;
    r.count_at = r.tiles_at + static_cast<size_t>(w.most_tiles) * sizeof(Tile);
    r.beyond_at = r.count_at + 16;
    ExpandGrid& g = r.grid;
    g.key_i = (a.n_heads * a.nope + 127) / 128;
    g.keys = g.key_i * ((a.n_rows + 127) / 128);
    g.value_i = static_cast<uint32_t>((w.value_rows + 127) / 128);
    g.values = g.value_i * ((a.n_heads * r.dv + 127) / 128);
    g.copies = 1024;
    r.bytes = r.beyond_at + (dtype == SVSX_F16 ? sizeof(uint4) * (static_cast<size_t>(g.keys) + g.values) : 0);
    return r;
}

template <typename T, int DK, int DV, int NW> hipError_t launch_prompt(const ExpandedArgs& a, const Space& w, const ExpandGrid& g, hipStream_t stream) {
    typedef PromptLayout<T, DK, DV, NW> L;
    static std::atomic<uint64_t> granted{0};
    if (const hipError_t e = grant_lds(reinterpret_cast<const void*>(prompt_kernel<T, DK, DV, NW>), L::kBytes, &granted); e != hipSuccess) return e;
    hipLaunchKernelGGL((prompt_kernel<T, DK, DV, NW>), dim3(w.most_tiles * a.n_heads), dim3(NW * 64), L::kBytes, stream, a, w, g);
    return hipGetLastError();
}

template <typename T> hipError_t launch_expanded(const ExpandedArgs& a, PromptRoute& r, void* workspace, hipStream_t stream) {
    if (!r.tiles) {
        hipLaunchKernelGGL(expanded_head_kernel<T>, dim3(std::min(a.n_heads * a.n_tokens, 1u << 20)), dim3(256), 0, stream, a); // a grid has fewer than 2^32 threads
        return hipGetLastError();
    }
    char* base = static_cast<char*>(workspace);
    Space& w = r.space;
    w.keys = base;
    w.values = base + r.values_at;
    w.tiles = reinterpret_cast<Tile*>(base + r.tiles_at);
    w.count = reinterpret_cast<uint32_t*>(base + r.count_at);
    w.beyond = reinterpret_cast<uint4*>(base + r.beyond_at);
    const ExpandGrid& g = r.grid;
    auto expand = r.wide ? expand_kernel<T, true> : expand_kernel<T, false>;
    hipLaunchKernelGGL(expand, dim3(g.keys + g.values + g.copies + 1), dim3(256), 0, stream, a, w, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || w.most_tiles == 0) return e;
    if constexpr (sizeof(T) == 2) {
        if (r.waves == 8) {
            if (r.dk == 128) return r.dv == 64 ? launch_prompt<T, 128, 64, 8>(a, w, g, stream) : launch_prompt<T, 128, 128, 8>(a, w, g, stream);
            return r.dv == 64 ? launch_prompt<T, 192, 64, 8>(a, w, g, stream) : launch_prompt<T, 192, 128, 8>(a, w, g, stream);
        }
    }
    if (r.dk == 128) return r.dv == 64 ? launch_prompt<T, 128, 64, 4>(a, w, g, stream) : launch_prompt<T, 128, 128, 4>(a, w, g, stream);
    if (r.dk == 192) return r.dv == 64 ? launch_prompt<T, 192, 64, 4>(a, w, g, stream) : launch_prompt<T, 192, 128, 4>(a, w, g, stream);
    return launch_prompt<T, 256, 256, 4>(a, w, g, stream);
}

} // namespace
} // namespace svsx

extern "C" {

int svsx_latent_expanded_workspace(const svsx_expanded_desc* desc, size_t* bytes) {
    ExpandedArgs a;
    if (const int rc = check_expanded(desc, &a)) return rc;
    if (!bytes) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *bytes = a.n_tokens ? route_of(a, desc->dtype).bytes : 0;
    return SVSX_SUCCESS;
}

int svsx_latent_expanded_device(const svsx_expanded_desc* desc, void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    ExpandedArgs a;
    if (const int rc = check_expanded(desc, &a)) return rc;
    if (a.n_tokens == 0) return SVSX_SUCCESS;
    PromptRoute r = route_of(a, desc->dtype);
    if (r.bytes > 0 && (!d_workspace || workspace_bytes < r.bytes || reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0))
        return fail(SVSX_INVALID_ARGUMENT, "a workspace of %zu bytes, aligned to 16, is needed", r.bytes);
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = desc->dtype == SVSX_F32   ? launch_expanded<float>(a, r, d_workspace, s)
                         : desc->dtype == SVSX_F16 ? launch_expanded<_Float16>(a, r, d_workspace, s)
                                                   : launch_expanded<bf16_t>(a, r, d_workspace, s);
    return e == hipSuccess ? SVSX_SUCCESS : fail(SVSX_RUNTIME_ERROR, "expanded attention launch failed: %s", hipGetErrorString(e));
}

} // extern "C"
