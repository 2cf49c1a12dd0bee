// svsx_attention.hip -- attention of one new token over paged rows (include/svsx.h: svsx_paged_attention_device).
#include "svsx_host.h"
#include "svsx_paged.h"

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
};

// rows of query i: its table row and how many rows there are
__device__ __forceinline__ uint32_t rows_of(const AttentionArgs& a, uint32_t i, const int32_t** table) {
    const int32_t s = a.sequences ? a.sequences[i] : static_cast<int32_t>(i);
    if (s < 0 || static_cast<uint32_t>(s) >= a.n_sequences) return 0;
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
    return SVSX_SUCCESS;
}

} // namespace
} // namespace svsx

extern "C" {

int svsx_paged_attention_workspace(const svsx_attention_desc* desc, size_t* bytes) {
    AttentionArgs a;
    if (const int rc = check_attention(desc, &a)) return rc;
    if (!bytes) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *bytes = 0;
    return SVSX_SUCCESS;
}

int svsx_paged_attention_device(const svsx_attention_desc* desc, void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    (void)d_workspace;
    (void)workspace_bytes;
    AttentionArgs a;
    if (const int rc = check_attention(desc, &a)) return rc;
    if (a.n_queries == 0) return SVSX_SUCCESS;
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    auto kernel = desc->dtype == SVSX_F32 ? attend_head_kernel<float> : desc->dtype == SVSX_F16 ? attend_head_kernel<_Float16> : attend_head_kernel<bf16_t>;
    hipLaunchKernelGGL(kernel, dim3(a.n_heads, a.n_queries), dim3(256), 0, static_cast<hipStream_t>(hip_stream), a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SVSX_SUCCESS : fail(SVSX_RUNTIME_ERROR, "attention launch failed: %s", hipGetErrorString(e));
}

} // extern "C"
