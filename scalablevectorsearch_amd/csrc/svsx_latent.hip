// svsx_latent.hip -- latent attention in its expanded form, for prompts (include/svsx.h: svsx_latent_expanded_device).
#include "svsx_host.h"
#include "svsx_paged.h"

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
};

// One workgroup per query and head, in the latent space: w_key applied to the query, w_value to the result.
template <typename T> __global__ __launch_bounds__(256) void expanded_head_kernel(const ExpandedArgs a) {
    __shared__ RowsShared sm;
    const uint32_t h = blockIdx.x, t = blockIdx.y;
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
    const size_t limit = size_t(1) << 31;
    if (d->n_tokens > 65535 * size_t(16) || d->n_rows >= limit || d->n_sequences >= limit) return fail(SVSX_INVALID_ARGUMENT, "too many queries, rows or sequences in one call");
    if (d->n_tokens > 0 && (!d->d_queries || !d->d_out || !d->d_w_value || (d->nope_dim > 0 && !d->d_w_key))) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    if (d->n_tokens > 0 && d->n_sequences > 0 && (!d->d_query_offsets || !d->d_row_offsets || (d->n_rows > 0 && !d->d_rows))) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *a = ExpandedArgs{d->d_queries, d->d_rows, d->d_w_key, d->d_w_value, d->d_query_offsets, d->d_row_offsets, d->d_out, d->query_stride, d->query_head_stride, d->row_stride,
                      static_cast<uint32_t>(d->n_sequences), static_cast<uint32_t>(d->n_tokens), static_cast<uint32_t>(d->n_rows), static_cast<uint32_t>(d->n_heads),
                      static_cast<uint32_t>(d->nope_dim), static_cast<uint32_t>(d->rope_dim), static_cast<uint32_t>(d->rank), static_cast<uint32_t>(d->value_dim), d->scale,
                      d->causal, d->keep_rest};
    return SVSX_SUCCESS;
}

} // namespace
} // namespace svsx

extern "C" {

int svsx_latent_expanded_workspace(const svsx_expanded_desc* desc, size_t* bytes) {
    ExpandedArgs a;
    if (const int rc = check_expanded(desc, &a)) return rc;
    if (!bytes) return fail(SVSX_INVALID_ARGUMENT, "null argument");
    *bytes = 0;
    return SVSX_SUCCESS;
}

int svsx_latent_expanded_device(const svsx_expanded_desc* desc, void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    (void)d_workspace;
    (void)workspace_bytes;
    ExpandedArgs a;
    if (const int rc = check_expanded(desc, &a)) return rc;
    if (a.n_tokens == 0) return SVSX_SUCCESS;
    if (a.n_tokens > 65535) return fail(SVSX_INVALID_ARGUMENT, "too many queries in one call");
    DeviceScope on(desc->device);
    if (on.error != hipSuccess) return fail(SVSX_RUNTIME_ERROR, "hipSetDevice(%d) failed: %s", desc->device, hipGetErrorString(on.error));
    auto kernel = desc->dtype == SVSX_F32 ? expanded_head_kernel<float> : desc->dtype == SVSX_F16 ? expanded_head_kernel<_Float16> : expanded_head_kernel<bf16_t>;
    hipLaunchKernelGGL(kernel, dim3(a.n_heads, a.n_tokens), dim3(256), 0, static_cast<hipStream_t>(hip_stream), a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SVSX_SUCCESS : fail(SVSX_RUNTIME_ERROR, "expanded attention launch failed: %s", hipGetErrorString(e));
}

} // extern "C"
