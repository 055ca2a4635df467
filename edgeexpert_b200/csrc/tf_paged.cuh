// tf_paged.cuh -- the paged KV cache as the kernels see it (tf_paged_kv), and the
// element types of the serving operators.
#pragma once
#include <type_traits>

#include "tf_context.cuh"

namespace tf {

constexpr int kMaxPagedHeadDim = 512;

// Device view of a tf_paged_kv: strides in elements, 64-bit, so a pool may be
// larger than 2^32 elements.
template <typename T>
struct PagedView {
    T* k;
    T* v;
    long long page_stride, pos_stride, head_stride;
    int num_pages, page_size;
};

template <typename T>
inline PagedView<T> paged_view(const tf_paged_kv* kv) {
    return {static_cast<T*>(kv->k),        static_cast<T*>(kv->v),   (long long)kv->page_stride,
            (long long)kv->position_stride, (long long)kv->head_stride, (int)kv->num_pages,
            (int)kv->page_size};
}

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// The checks that every entry point taking a tf_paged_kv makes.
inline tf_status check_paged_kv(tf_context* ctx, const tf_paged_kv* kv, const char* name) {
    if (!kv || !kv->k || !kv->v) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null cache", name);
    if (kv->num_pages == 0 || kv->page_size == 0 || kv->num_kv_heads == 0)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: empty cache", name);
    if ((uint64_t)kv->num_pages * kv->page_size > 0x7FFFFFFFull)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: num_pages * page_size must be below 2^31", name);
    if (kv->head_dim == 0 || kv->head_dim % 8 || kv->head_dim > (uint32_t)kMaxPagedHeadDim)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: head_dim must be a multiple of 8 up to %d", name,
                    kMaxPagedHeadDim);
    if (kv->dtype != TF_DTYPE_F16 && kv->dtype != TF_DTYPE_BF16)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: unknown cache dtype", name);
    // a row of one head must not run into the next head, position or page
    if (kv->page_stride % 8 || kv->position_stride % 8 || kv->head_stride % 8 || !aligned16(kv->k) ||
        !aligned16(kv->v))
        return fail(ctx, TF_ERR_MISALIGNED, "%s: cache pointers 16-byte aligned, strides multiples of 8", name);
    if ((kv->num_kv_heads > 1 && kv->head_stride < kv->head_dim) ||
        (kv->page_size > 1 && kv->position_stride < kv->head_dim) ||
        (kv->num_pages > 1 && kv->page_stride < kv->head_dim))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: cache strides below head_dim", name);
    return TF_OK;
}

// A launch whose start-up overlaps the end of what is before it in the stream (the kernels
// wait for that before they read anything).
template <typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Args...), unsigned ctas, unsigned threads, size_t smem, cudaStream_t cs,
                              const std::common_type_t<Args>&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent_launches() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline tf_status enter(tf_context* ctx, const char* name) {
    if (!ctx) return TF_ERR_INVALID_ARG;
    if (cudaSetDevice(ctx->device) != cudaSuccess) return fail(ctx, TF_ERR_CUDA, "%s: cudaSetDevice failed", name);
    return TF_OK;
}

}  // namespace tf
