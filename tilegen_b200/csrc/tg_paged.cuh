// Shared pieces of the paged operators (tg_rope.cu, tg_paged_host.cu, tg_prefix_attn*.cu):
// 16-bit conversions, the CSR page-table lookup and the host-side checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "../../include/tilegen_b200_paged.h"
#include "tg_common.cuh"

namespace tg {

constexpr int kSMs = 148;  // B200: two dies of 74

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two numbers in one word of a 16-bit type, and back.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    } else {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}

// The sequence that token t belongs to: the last b with q_indptr[b] <= t, clamped to a
// sequence (token b is sequence b's where there is no q_indptr).
__device__ __forceinline__ int64_t sequence_of(const int64_t* q_indptr, int64_t rows, int64_t t) {
    if (!q_indptr) return t;
    int64_t lo = 0, hi = rows;  // q_indptr[lo] <= t
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (q_indptr[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same for a token that is the same in all lanes of a full warp: 32 places at a time, so that
// a batch of 1024 takes two loads one after the other instead of ten.
__device__ __forceinline__ int64_t sequence_of_warp(const int64_t* q_indptr, int rows, int t) {
    if (!q_indptr) return t;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = rows;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const uint32_t below = __ballot_sync(kFull, at < n && q_indptr[lo + at] <= t);
        const int k = below ? 31 - __clz(below) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// First token and number of tokens of sequence b, inside [0, tokens] whatever q_indptr holds.
__device__ __forceinline__ void tokens_of(const int64_t* q_indptr, int64_t tokens, int64_t b, int64_t& first,
                                          int64_t& n) {
    if (!q_indptr) {
        first = b;
        n = 1;
        return;
    }
    const int64_t a = q_indptr[b], e = q_indptr[b + 1];
    first = min(max(a, (int64_t)0), tokens);
    n = min(max(e, first), tokens) - first;
}

// Pages of row b of the table inside [0, nnz] whatever indptr holds.
__device__ __forceinline__ void pages_of(const int64_t* indptr, int64_t nnz, int64_t b, int64_t& first, int64_t& n) {
    const int64_t a = indptr[b], e = indptr[b + 1];
    first = min(max(a, (int64_t)0), nnz);
    n = min(max(e, first), nnz) - first;
}

// The stride of a dimension of n: nothing is multiplied by that of a dimension of one, which may be
// anything and must not decide how rows are moved or whether they are refused.
inline int64_t stride_of(int64_t n, int64_t stride) { return n > 1 ? stride : 0; }

// host side (tg_paged_host.cu)
int check_cache(const tg_paged_kv* c, const char* op);
int check_table(const tg_csr* t, const tg_paged_kv* c, int64_t tokens, const int64_t* q_indptr, const int64_t* seq_len,
                const char* op);
int check_rope(const tg_rope* r, int32_t dim, const char* op);
// Synchronous check of the index arrays on `st` (TG_FLAG_BOUNDS_CHECK).
int paged_bounds_check(const tg_csr& t, int64_t page_size, const int64_t* seq_len, int64_t max_seq_len, int64_t tokens,
                       const int64_t* q_indptr, int64_t max_q_len, const int64_t* prefix_pages, int64_t n_prefix,
                       bool append, const char* op, cudaStream_t st);
// Raises a kernel's limit of dynamic shared memory, once on each device.
struct SmemOnce {
    std::atomic<uint64_t> done{0};  // devices, by bit
    int raise(const void* kernel, int bytes) {
        int dev = 0;
        const int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
        if (rc != TG_OK || (dev < 64 && done.load(std::memory_order_relaxed) >> dev & 1)) return rc;
        const int set = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                                   "cudaFuncSetAttribute");
        if (set == TG_OK && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
        return set;
    }
};

// Launch with the programmatic-dependency attribute: the kernel may start while the one
// before it on the stream still runs, and orders itself with pdl_wait().
template <typename... P, typename... A>
int launch_pdl(const char* what, void (*kernel)(P...), dim3 grid, int block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    const int rc = check_launch(what);
    return e != cudaSuccess ? check_cuda(e, what) : rc;
}

}  // namespace tg
