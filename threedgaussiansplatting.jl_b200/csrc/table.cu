// table.cu — rows of SH coefficients shared through a table.
//   gs3d_table_lookup    out[i] = scale * table[indices[i]]
//   gs3d_table_gradient  table_grads[k] = scale * sum of grads[f] over the rows f with index k + 1,
//                        by the rows sorted by index (stable), so the order of every sum is fixed
#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace gs3d {
namespace {

int grid_for(int64_t items, int threads, int per_sm) {
    const int64_t b = std::min<int64_t>(ceil_div(items, threads), (int64_t)device_sm_count() * per_sm);
    return (int)std::max<int64_t>(b, 1);
}

template <typename TI, typename TO>
__global__ void __launch_bounds__(256) k_table_lookup(const TI* __restrict__ table, int64_t rows,
                                                      int64_t table_stride, const int32_t* __restrict__ indices,
                                                      float scale, TO* __restrict__ out, int64_t n,
                                                      int64_t out_stride, int dim) {
    const int64_t total = n * dim;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / dim;
        const int c = (int)(i - r * dim);
        const int k = indices[r];
        float v = 0.0f;
        if (k >= 1 && k <= rows) v = to_f32(table[(int64_t)(k - 1) * table_stride + c]) * scale;
        out[r * out_stride + c] = from_f32<TO>(v);
    }
}

// ---- gradient --------------------------------------------------------------------------------
// Row f's key: its table row 1 .. rows, or 0 where it takes no part.
__global__ void __launch_bounds__(256) k_table_keys(const int32_t* __restrict__ indices, int64_t n_indices,
                                                    const int32_t* __restrict__ f2g,
                                                    const int32_t* __restrict__ counts, int64_t n, int64_t rows,
                                                    int64_t* __restrict__ keys, int32_t* __restrict__ vals) {
    const int64_t live = counts ? min((int64_t)max(counts[0], 0), n) : n;
    for (int64_t f = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; f < n;
         f += (int64_t)gridDim.x * blockDim.x) {
        int k = 0;
        if (f < live) {
            const int64_t i = f2g ? (int64_t)f2g[f] - 1 : f;
            if (i >= 0 && i < n_indices) k = indices[i];
            if (k < 1 || k > rows) k = 0;
        }
        keys[f] = k;
        vals[f] = (int32_t)f;
    }
}

__device__ __forceinline__ int64_t first_not_below(const int64_t* keys, int64_t n, int64_t k) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < k) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// One block per table row: threads side by side on the columns, `slots` of them one after the other
// on the rows of the segment; the slots' sums are added in order.
template <typename T>
__global__ void __launch_bounds__(128) k_table_reduce(const T* __restrict__ grads, int64_t stride, int dim,
                                                      const int64_t* __restrict__ keys,
                                                      const int32_t* __restrict__ vals, int64_t n, float scale,
                                                      float* __restrict__ out, int64_t out_stride, int accumulate) {
    __shared__ int64_t seg[2];
    __shared__ float part[128];
    const int64_t k = blockIdx.x;
    if (threadIdx.x < 2) seg[threadIdx.x] = first_not_below(keys, n, k + 1 + threadIdx.x);
    __syncthreads();
    const int wide = min(dim, 128), slots = 128 / wide;
    const int slot = threadIdx.x / wide, col = threadIdx.x - slot * wide;
    for (int c0 = 0; c0 < dim; c0 += wide) {
        const int c = c0 + col;
        float s = 0.0f;
        if (slot < slots && c < dim)
            for (int64_t j = seg[0] + slot; j < seg[1]; j += slots) s += to_f32(grads[(int64_t)vals[j] * stride + c]);
        part[threadIdx.x] = s;
        __syncthreads();
        if (slot == 0 && c < dim) {
            for (int q = 1; q < slots; ++q) s += part[q * wide + col];
            float* o = out + k * out_stride + c;
            *o = accumulate ? *o + scale * s : scale * s;
        }
        __syncthreads();
    }
}

struct GradLayout {
    size_t keys, vals, skeys, svals, sort, total;
};

GradLayout grad_layout(int64_t n) {
    GradLayout L;
    size_t off = 0;
    L.keys = off; off += align256((size_t)n * 8);
    L.vals = off; off += align256((size_t)n * 4);
    L.skeys = off; off += align256((size_t)n * 8);
    L.svals = off; off += align256((size_t)n * 4);
    L.sort = off; off += radix_sort_workspace_bytes(n);
    L.total = off;
    return L;
}

int bits_of(int64_t v) {
    int b = 0;
    while (v >> b) ++b;
    return b;
}

}  // namespace
}  // namespace gs3d

using namespace gs3d;

extern "C" {

GS3D_API int gs3d_table_lookup(const gs3d_rows* table, const int32_t* indices, float scale, const gs3d_rows* out,
                               gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(table, "table"));
    GS3D_RETURN_IF(check_rows(out, "lookup output"));
    if (table->dim != out->dim) return invalid("table dim %d, output dim %d", table->dim, out->dim);
    if (out->rows == 0) return GS3D_OK;
    if (!indices) return invalid("NULL indices");
    ProfScope prof("table_lookup", stream);
    return dispatch_type(table->type, [&](auto ti) {
        using TI = typename decltype(ti)::T;
        return dispatch_type(out->type, [&](auto to) {
            using TO = typename decltype(to)::T;
            k_table_lookup<TI, TO><<<grid_for(out->rows * out->dim, 256, 8), 256, 0, stream>>>(
                static_cast<const TI*>(table->data), table->rows, table->row_stride, indices, scale,
                static_cast<TO*>(out->data), out->rows, out->row_stride, out->dim);
            GS3D_LAUNCHED("k_table_lookup");
            return GS3D_OK;
        });
    });
}

GS3D_API int gs3d_table_gradient_workspace_size(int64_t grad_rows, int64_t table_rows, int32_t dim, size_t* bytes) {
    if (!bytes) return invalid("bytes is NULL");
    if (grad_rows < 0 || grad_rows > kMaxRows || table_rows < 0 || table_rows > kMaxRows || dim < 1 ||
        dim > kMaxRowDim)
        return invalid("%lld rows, table of %lld rows, dim %d", (long long)grad_rows, (long long)table_rows, dim);
    *bytes = grad_layout(std::max<int64_t>(grad_rows, 1)).total;
    return GS3D_OK;
}

GS3D_API int gs3d_table_gradient(const gs3d_rows* grads, const int32_t* indices, int64_t n_indices,
                                 const int32_t* fgidx_to_gidx, const int32_t* device_counts, float scale,
                                 const gs3d_rows* table_grads, uint32_t flags, void* workspace,
                                 size_t workspace_bytes, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(grads, "gradients"));
    GS3D_RETURN_IF(check_rows(table_grads, "table gradients"));
    if (grads->dim != table_grads->dim)
        return invalid("gradient dim %d, table dim %d", grads->dim, table_grads->dim);
    if (table_grads->type != GS3D_F32) return invalid("table gradients are GS3D_F32");
    if (flags & ~GS3D_TABLE_ACCUMULATE) return invalid("flags %u", flags);
    if (n_indices < 0 || (!fgidx_to_gidx && n_indices < grads->rows))
        return invalid("%lld indices for %lld rows", (long long)n_indices, (long long)grads->rows);
    if (grads->rows > 0 && !indices && n_indices > 0) return invalid("NULL indices");
    if (table_grads->rows == 0) return GS3D_OK;
    const int64_t n = grads->rows;
    const GradLayout L = grad_layout(std::max<int64_t>(n, 1));
    if (!workspace || workspace_bytes < L.total)
        return set_error("table gradient workspace %zu bytes < %zu", workspace_bytes, L.total), GS3D_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return invalid("workspace not 256-byte aligned");
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    int64_t* keys = reinterpret_cast<int64_t*>(ws + L.keys);
    int32_t* vals = reinterpret_cast<int32_t*>(ws + L.vals);
    int64_t* skeys = reinterpret_cast<int64_t*>(ws + L.skeys);
    int32_t* svals = reinterpret_cast<int32_t*>(ws + L.svals);
    ProfScope prof("table_grad", stream);
    if (n > 0) {
        k_table_keys<<<grid_for(n, 256, 8), 256, 0, stream>>>(indices, n_indices, fgidx_to_gidx, device_counts, n,
                                                              table_grads->rows, keys, vals);
        GS3D_LAUNCHED("k_table_keys");
        GS3D_RETURN_IF(radix_sort_pairs(ws + L.sort, L.total - L.sort, keys, skeys, vals, svals, n, nullptr, n,
                                        bits_of(table_grads->rows), stream));
    }
    return dispatch_type(grads->type, [&](auto t) {
        using T = typename decltype(t)::T;
        k_table_reduce<T><<<(unsigned)table_grads->rows, 128, 0, stream>>>(
            static_cast<const T*>(grads->data), grads->row_stride, grads->dim, skeys, svals, n, scale,
            static_cast<float*>(table_grads->data), table_grads->row_stride, (flags & GS3D_TABLE_ACCUMULATE) ? 1 : 0);
        GS3D_LAUNCHED("k_table_reduce");
        return GS3D_OK;
    });
}

}  // extern "C"
