// Argument and index checks shared by the paged operators.
#include <algorithm>

#include "tg_prefix_attn.cuh"
#include "tg_rope.cuh"

namespace tg {

int check_cache(const tg_paged_kv* c, const char* op) {
    if (!c) return set_error(TG_EINVAL, "%s: null cache descriptor", op);
    if (c->pages < 0 || c->page_size < 1 || c->heads < 1 || c->dim < 1)
        return set_error(TG_EINVAL, "%s: bad cache (pages=%lld page_size=%lld heads=%d dim=%d)", op,
                         (long long)c->pages, (long long)c->page_size, c->heads, c->dim);
    if (c->pages > INT32_MAX || c->page_size > INT32_MAX)
        return set_error(TG_EINVAL, "%s: page numbers and slots are 32-bit (pages=%lld page_size=%lld)", op,
                         (long long)c->pages, (long long)c->page_size);
    if (c->pages > 0 && (!c->k || !c->v)) return set_error(TG_EINVAL, "%s: null cache", op);
    return TG_OK;
}

int check_table(const tg_csr* t, const tg_paged_kv* c, int64_t tokens, const int64_t* q_indptr, const int64_t* seq_len,
                const char* op) {
    if (!t) return set_error(TG_EINVAL, "%s: null page table", op);
    if (t->rows < 0 || t->nnz < 0 || tokens < 0)
        return set_error(TG_EINVAL, "%s: negative size (sequences=%lld pages=%lld tokens=%lld)", op,
                         (long long)t->rows, (long long)t->nnz, (long long)tokens);
    if (t->cols != c->pages)
        return set_error(TG_EINVAL, "%s: the page table has %lld columns and the cache %lld pages", op,
                         (long long)t->cols, (long long)c->pages);
    if (t->rows > INT32_MAX || tokens > INT32_MAX)
        return set_error(TG_EINVAL, "%s: more than 2^31 sequences or tokens", op);
    if (!q_indptr && tokens != t->rows)
        return set_error(TG_EINVAL, "%s: %lld tokens for %lld sequences need a q_indptr", op, (long long)tokens,
                         (long long)t->rows);
    if (tokens > 0 && t->rows == 0) return set_error(TG_EINVAL, "%s: tokens without a sequence", op);
    if (tokens > 0 && (!t->indptr || !seq_len)) return set_error(TG_EINVAL, "%s: null indptr/seq_len", op);
    if (t->nnz > 0 && !t->indices) return set_error(TG_EINVAL, "%s: null page indices", op);
    return TG_OK;
}

int check_rope(const tg_rope* r, int32_t dim, const char* op) {
    if (r->rot_dim < 0 || r->rot_dim > dim || r->rot_dim % 2)
        return set_error(TG_EINVAL, "%s: rot_dim must be even and in [0, %d] (got %d)", op, dim, r->rot_dim);
    if (r->layout != TG_ROPE_HALF && r->layout != TG_ROPE_INTERLEAVED)
        return set_error(TG_EINVAL, "%s: layout must be TG_ROPE_HALF or TG_ROPE_INTERLEAVED (got %d)", op, r->layout);
    if (r->rot_dim > 0 && !r->freq) return set_error(TG_EINVAL, "%s: null freq", op);
    return TG_OK;
}

namespace {

// Sets bits of *err: 1 indptr[0] != 0, 2 indptr decreasing, 4 indptr[rows] != nnz, 8 page
// number outside the cache, 16 a length outside [0, min(its pages' slots, max_seq_len)],
// 32 q_indptr not 0 .. tokens without a step back or with more than max_q_len tokens in a
// sequence, 64 prefix page outside the cache, 128 more new tokens than the sequence is long.
__global__ void paged_check_kernel(tg_csr t, int64_t page_size, const int64_t* seq_len, int64_t max_seq_len,
                                   int64_t tokens, const int64_t* q_indptr, int64_t max_q_len,
                                   const int64_t* prefix_pages, int64_t n_prefix, bool append, uint32_t* err) {
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    uint32_t e = 0;
    if (tid == 0) {
        if (t.indptr[0] != 0) e |= 1u;
        if (t.indptr[t.rows] != t.nnz) e |= 4u;
        if (q_indptr && (q_indptr[0] != 0 || q_indptr[t.rows] != tokens)) e |= 32u;
    }
    for (int64_t b = tid; b < t.rows; b += stride) {
        const int64_t pages = t.indptr[b + 1] - t.indptr[b], len = seq_len[b];
        if (pages < 0) e |= 2u;
        if (len < 0 || len > max_seq_len || ceil_div(len, page_size) > pages) e |= 16u;
        const int64_t n = q_indptr ? q_indptr[b + 1] - q_indptr[b] : 1;
        if (n < 0 || n > max_q_len) e |= 32u;
        if (append && n > len) e |= 128u;
    }
    for (int64_t p = tid; p < t.nnz; p += stride)
        if (t.indices[p] < 0 || t.indices[p] >= t.cols) e |= 8u;
    for (int64_t p = tid; p < n_prefix; p += stride)
        if (prefix_pages[p] < 0 || prefix_pages[p] >= t.cols) e |= 64u;
    if (e) atomicOr(err, e);
}

}  // namespace

int paged_bounds_check(const tg_csr& t, int64_t page_size, const int64_t* seq_len, int64_t max_seq_len, int64_t tokens,
                       const int64_t* q_indptr, int64_t max_q_len, const int64_t* prefix_pages, int64_t n_prefix,
                       bool append, const char* op, cudaStream_t st) {
    if (t.rows == 0) return TG_OK;
    CheckWord word;
    int rc = word.take();
    if (rc != TG_OK) return rc;
    uint32_t* const err = word.at;
    rc = check_cuda(cudaMemsetAsync(err, 0, sizeof(uint32_t), st), "cudaMemsetAsync");
    if (rc != TG_OK) return rc;
    const int64_t blocks = std::min<int64_t>(ceil_div(std::max({t.rows, t.nnz, n_prefix}) + 1, 256), kSMs * 16);
    paged_check_kernel<<<(unsigned)blocks, 256, 0, st>>>(t, page_size, seq_len, max_seq_len, tokens, q_indptr,
                                                         max_q_len, prefix_pages, n_prefix, append, err);
    rc = check_launch("paged_check_kernel");
    if (rc != TG_OK) return rc;
    uint32_t h = 0;
    rc = check_cuda(cudaMemcpyAsync(&h, err, sizeof(h), cudaMemcpyDeviceToHost, st), "cudaMemcpyAsync");
    if (rc != TG_OK) return rc;
    rc = check_cuda(cudaStreamSynchronize(st), "cudaStreamSynchronize");
    if (rc != TG_OK) return rc;
    if (h)
        return set_error(TG_EBOUNDS, "%s: index check failed (flags 0x%x:%s%s%s%s%s%s%s%s)", op, h,
                         (h & 1) ? " indptr[0]!=0" : "", (h & 2) ? " indptr decreasing" : "",
                         (h & 4) ? " indptr[rows]!=nnz" : "", (h & 8) ? " page out of range" : "",
                         (h & 16) ? " seq_len out of range" : "", (h & 32) ? " q_indptr" : "",
                         (h & 64) ? " prefix page out of range" : "", (h & 128) ? " more new tokens than seq_len" : "");
    return TG_OK;
}

int check_append(const tg_kv_append_args* a, const char* op, cudaStream_t st, bool& done) {
    done = false;
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_cache(a->cache, op);
    if (rc == TG_OK) rc = check_table(a->pages, a->cache, a->tokens, a->q_indptr, a->seq_len, op);
    if (rc == TG_OK && a->rope) rc = check_rope(a->rope, a->cache->dim, op);
    if (rc == TG_OK && a->rope) rc = check_rot(a->rope, op);
    if (rc != TG_OK) return rc;
    if (a->flags & ~TG_FLAG_BOUNDS_CHECK) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if (a->q && (!a->q_out || a->q_heads < 0)) return set_error(TG_EINVAL, "%s: q without q_out, or q_heads < 0", op);
    if (a->tokens == 0) {
        done = true;
        return TG_OK;
    }
    if (!a->k.data || !a->v.data) return set_error(TG_EINVAL, "%s: null k/v", op);
    if (a->q && a->q_heads > 0 && (!a->q->data || !a->q_out->data)) return set_error(TG_EINVAL, "%s: null q/q_out", op);
    if (a->flags & TG_FLAG_BOUNDS_CHECK)
        return paged_bounds_check(*a->pages, a->cache->page_size, a->seq_len, INT64_MAX, a->tokens, a->q_indptr, INT64_MAX,
                                  nullptr, 0, true, op, st);
    return TG_OK;
}

// ------------------------------------------------------------------ tensor maps
namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

}  // namespace

int cache_maps(const AttnParams& p, bool is_half, int dim, int box_rows, CUtensorMap* k, CUtensorMap* v) {
    *k = *v = CUtensorMap{};
    if (p.pages == 0) return TG_OK;  // no page, no box
    if (!encoder()) return set_error(TG_ECUDA, "cuTensorMapEncodeTiled is not available");
    // the stride of a dimension of one is of no use to anyone and may be anything
    const auto bytes = [&](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 ? stride : dim) * 2; };
    for (int i = 0; i < 2; ++i) {
        const int64_t page = i ? p.v_page : p.k_page, slot = i ? p.v_slot : p.k_slot, head = i ? p.v_head : p.k_head;
        const cuuint64_t size[4] = {(cuuint64_t)dim, (cuuint64_t)p.page_size, (cuuint64_t)p.kv_heads, (cuuint64_t)p.pages};
        const cuuint64_t stride[3] = {bytes(p.page_size, slot), bytes(p.kv_heads, head), bytes(p.pages, page)};
        const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
        const CUresult r = encoder()(i ? v : k, is_half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                                     const_cast<void*>(i ? p.v : p.k), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS)
            return set_error(TG_ECUDA, "cuTensorMapEncodeTiled: CUDA error %d (page_size=%d strides %lld %lld %lld)", (int)r,
                             p.page_size, (long long)page, (long long)slot, (long long)head);
    }
    return TG_OK;
}

int rows_map(const AttnParams& p, bool is_half, int dim, int box_heads, int box_tokens, CUtensorMap* q) {
    *q = CUtensorMap{};
    if (p.tokens == 0) return TG_OK;  // no token, no box
    if (!encoder()) return set_error(TG_ECUDA, "cuTensorMapEncodeTiled is not available");
    const auto bytes = [&](int64_t n, int64_t stride) { return (cuuint64_t)(n > 1 ? stride : dim) * 2; };
    const cuuint64_t size[3] = {(cuuint64_t)dim, (cuuint64_t)p.q_heads, (cuuint64_t)p.tokens};
    const cuuint64_t stride[2] = {bytes(p.q_heads, p.q_head), bytes(p.tokens, p.q_tok)};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, step[3] = {1, 1, 1};
    const CUresult r = encoder()(q, is_half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                                 const_cast<void*>(p.q), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(TG_ECUDA, "cuTensorMapEncodeTiled: CUDA error %d (queries, strides %lld %lld)", (int)r,
                         (long long)p.q_head, (long long)p.q_tok);
    return TG_OK;
}

}  // namespace tg
