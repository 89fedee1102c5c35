// Rotary positions and the paged-cache append (tg_rope_*, tg_kv_append_*).
//
// Pair i of a head's rotating elements (a, b) becomes scale * (a cos t - b sin t,
// b cos t + a sin t) with t = position * freq[i]; the gradient is the same with -t.  One
// kernel serves both calls: its rows are the heads of a token, of three kinds -- q (rotated
// into an output), k (rotated into the token's cache slot) and v (copied there).
//
// * Bound: HBM.  Each element is read once and written once, 16 bytes a load, and the
//   angles cost no traffic: a CTA takes a few tokens, computes their cosines and sines once
//   into shared memory, and all heads of these tokens use them.
// * The angle and its rest after whole turns (2 pi in two parts, after Cody and Waite) are
//   64-bit, so a position of 1e6 is as exact as position 1; the sine and cosine of the rest,
//   the rotation itself and its sum are 32-bit, rounded once to the output's type.
#include <algorithm>

#include "tg_paged.cuh"

namespace tg {
namespace {

template <typename T>
struct RopeParams {
    // q, k, v rows: input and output with their token and head strides (k and v go to the
    // slot offset of the token instead of a token stride)
    const T *q, *k, *v;
    T *qo, *ko, *vo;
    int64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, ko_page, ko_slot, ko_head, v_tok, v_head, vo_page, vo_slot,
        vo_head;
    int q_rows, kv_rows;  // heads
    int dim, rot;
    const double* freq;
    float scale, sign;
    int64_t tokens;
    int tile;  // tokens of a CTA
    const int64_t* positions;
    // append only
    int64_t position_base;
    const int64_t *q_indptr, *seq_len, *indptr, *indices;
    int64_t rows, pages, nnz, page_size;
    int lanes;  // threads along a row
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

constexpr int kRopeThreads = 256;
constexpr int kRopeTile = 32;         // most tokens of a CTA
constexpr int kRopeSmem = 32 * 1024;  // most bytes of cosines and sines of a CTA

// VEC elements are moved at once: 16 bytes where rows, strides and the parts of a row are
// multiples of that, else single elements.
template <typename T, int VEC, bool HALF, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams<T> p) {
    extern __shared__ float2 s_turn[];  // [tile][pairs] scale * (cos, sin)
    __shared__ double s_pos[kRopeTile];
    __shared__ int64_t s_page[kRopeTile];  // the token's cache page, -1: no such slot
    __shared__ int64_t s_slot[kRopeTile];
    using P = Pack<T, VEC>;
    const int tid = threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * p.tile;
    const int tile = (int)min((int64_t)p.tile, p.tokens - t0);
    if (tid < tile) {
        const int64_t t = t0 + tid;
        if constexpr (APPEND) {
            const int64_t b = sequence_of(p.q_indptr, p.rows, t);
            int64_t first, n, page0, npages;
            tokens_of(p.q_indptr, p.tokens, b, first, n);
            pages_of(p.indptr, p.nnz, b, page0, npages);
            const int64_t at = p.seq_len[b] - n + (t - first);
            int64_t page = -1;
            if (at >= 0 && t >= first && t < first + n) {
                const int64_t j = at / p.page_size;
                if (j < npages) page = p.indices[page0 + j];
                if (page >= p.pages) page = -1;
                s_slot[tid] = at - j * p.page_size;
            }
            s_page[tid] = page;
            s_pos[tid] = (double)(p.positions ? p.positions[t] : p.position_base + at);
        } else {
            s_pos[tid] = (double)p.positions[t];
        }
    }
    __syncthreads();
    const int pairs = p.rot / 2;
    for (int i = tid; i < tile * pairs; i += blockDim.x) {
        const int tt = i / pairs;
        const double t = s_pos[tt] * p.freq[i - tt * pairs];
        const double k = rint(t * 0.15915494309189533577);  // whole turns
        const double rest = fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, t));  // 2 pi in two parts
        float s, c;
        sincospif((float)(rest * 0.31830988618379067154), &s, &c);
        s_turn[i] = make_float2(c * p.scale, s * p.scale * p.sign);
    }
    __syncthreads();

    const int rows = p.q_rows + (APPEND ? 2 * p.kv_rows : 0);
    const int lane = tid % p.lanes, step = blockDim.x / p.lanes;
    const int turning = pairs / VEC;                         // chunks of pairs in a row
    const int chunks = turning + (p.dim - p.rot) / VEC;      // and of copied elements behind them
    int tt = 0, row = tid / p.lanes;
    for (;; row += step) {
        while (row >= rows) {
            row -= rows;
            ++tt;
        }
        if (tt >= tile) break;
        const T* in;
        T* out;
        const int64_t t = t0 + tt;
        if (!APPEND || row < p.q_rows) {
            in = p.q + t * p.q_tok + row * p.q_head;
            out = p.qo + t * p.qo_tok + row * p.qo_head;
        } else {
            const int64_t page = s_page[tt];
            if (page < 0) continue;
            const int h = row - p.q_rows;
            if (h >= p.kv_rows) {
                in = p.v + t * p.v_tok + (h - p.kv_rows) * p.v_head;
                out = p.vo + page * p.vo_page + s_slot[tt] * p.vo_slot + (h - p.kv_rows) * p.vo_head;
                for (int c = lane; c < p.dim / VEC; c += p.lanes)
                    reinterpret_cast<P*>(out)[c] = reinterpret_cast<const P*>(in)[c];
                continue;
            }
            in = p.k + t * p.k_tok + h * p.k_head;
            out = p.ko + page * p.ko_page + s_slot[tt] * p.ko_slot + h * p.ko_head;
        }
        const float2* turn = s_turn + tt * pairs;
        for (int c = lane; c < chunks; c += p.lanes) {
            if (c >= turning) {
                const int at = p.rot / VEC + c - turning;
                reinterpret_cast<P*>(out)[at] = reinterpret_cast<const P*>(in)[at];
                continue;
            }
            // two packs hold VEC pairs: halves apart, or neighbours
            const int ia = HALF ? c : 2 * c, ib = HALF ? turning + c : 2 * c + 1;
            P a = reinterpret_cast<const P*>(in)[ia], b = reinterpret_cast<const P*>(in)[ib];
            float x[2 * VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                x[j] = to_f32(a.v[j]);
                x[VEC + j] = to_f32(b.v[j]);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float2 cs = turn[c * VEC + j];
                const int k0 = HALF ? j : 2 * j, k1 = HALF ? VEC + j : 2 * j + 1;
                const float u = x[k0], w = x[k1];
                x[k0] = u * cs.x - w * cs.y;
                x[k1] = w * cs.x + u * cs.y;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a.v[j] = from_f32<T>(x[j]);
                b.v[j] = from_f32<T>(x[VEC + j]);
            }
            reinterpret_cast<P*>(out)[ia] = a;
            reinterpret_cast<P*>(out)[ib] = b;
        }
    }
}

template <typename T, bool APPEND>
int rope_run(RopeParams<T> p, int layout, cudaStream_t st, const char* what) {
    if (p.tokens == 0 || p.dim == 0) return TG_OK;
    constexpr int WIDE = 16 / (int)sizeof(T);
    // every address and stride in bytes, or'ed into one word: aligned where all of them are
    const void* const at[] = {p.q, p.qo, p.k, p.ko, p.v, p.vo};
    const int64_t strides[] = {p.q_tok,  p.q_head,  p.qo_tok,  p.qo_head, p.k_tok,  p.k_head,  p.ko_page,
                               p.ko_slot, p.ko_head, p.v_tok,  p.v_head,  p.vo_page, p.vo_slot, p.vo_head};
    uint64_t all = 0;
    for (const void* a : at) all |= reinterpret_cast<uint64_t>(a);
    for (const int64_t s : strides) all |= (uint64_t)s * sizeof(T);
    const bool wide = all % 16 == 0 && p.rot % (2 * WIDE) == 0 && (p.dim - p.rot) % WIDE == 0;
    const int vec = wide ? WIDE : 1;
    const int chunks = (p.rot / 2 + p.dim - p.rot) / vec;
    p.lanes = std::min(chunks, kRopeThreads);
    const int rows = p.q_rows + (APPEND ? 2 * p.kv_rows : 0);
    const int block = p.lanes * std::min(kRopeThreads / p.lanes, std::max(rows, 1) * kRopeTile);
    // Tokens of a CTA: enough that each thread moves a few rows for its share of the sines, but
    // at least eight CTAs an SM (a few tokens are one CTA each).
    const int pairs = p.rot / 2;
    int64_t tile = ceil_div(4ll * (block / p.lanes), std::max(rows, 1));
    tile = std::min<int64_t>({tile, kRopeTile, std::max<int64_t>(1, p.tokens / (kSMs * 8)),
                              pairs ? std::max<int64_t>(1, kRopeSmem / (pairs * 8)) : kRopeTile});
    p.tile = (int)tile;
    const size_t smem = (size_t)tile * pairs * sizeof(float2);
    const unsigned grid = (unsigned)ceil_div(p.tokens, tile);
    const bool half = layout == TG_ROPE_HALF;
    auto kernel = wide ? (half ? rope_kernel<T, WIDE, true, APPEND> : rope_kernel<T, WIDE, false, APPEND>)
                       : (half ? rope_kernel<T, 1, true, APPEND> : rope_kernel<T, 1, false, APPEND>);
    kernel<<<grid, block, smem, st>>>(p);
    return check_launch(what);
}

constexpr int kMaxRot = 2 * (kRopeSmem / 8);  // one token's cosines and sines fit a CTA

int check_rot(const tg_rope* r, const char* op) {
    return r->rot_dim > kMaxRot ? set_error(TG_EUNSUPPORTED, "%s: rot_dim above %d", op, kMaxRot) : TG_OK;
}

template <typename T>
int rope(const tg_rope* r, const tg_rows* x, const tg_rows* y, int64_t tokens, int32_t heads, int32_t dim,
         const int64_t* positions, uint32_t flags, tg_stream_t stream, const char* op) {
    if (!r || !x || !y) return set_error(TG_EINVAL, "%s: null descriptor", op);
    if (tokens < 0 || heads < 0 || dim < 0 || tokens > INT32_MAX)
        return set_error(TG_EINVAL, "%s: bad size (tokens=%lld heads=%d dim=%d)", op, (long long)tokens, heads, dim);
    if (flags & ~TG_FLAG_ROPE_INVERSE) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, flags);
    int rc = check_rope(r, dim, op);
    if (rc == TG_OK) rc = check_rot(r, op);
    if (rc != TG_OK) return rc;
    if (tokens == 0 || heads == 0 || dim == 0) return TG_OK;
    if (!x->data || !y->data) return set_error(TG_EINVAL, "%s: null x/y", op);
    if (!positions) return set_error(TG_EINVAL, "%s: null positions", op);
    RopeParams<T> p = {};
    p.q = static_cast<const T*>(x->data);
    p.qo = static_cast<T*>(y->data);
    p.q_tok = x->token_stride, p.q_head = x->head_stride;
    p.qo_tok = y->token_stride, p.qo_head = y->head_stride;
    p.q_rows = heads;
    p.dim = dim, p.rot = r->rot_dim;
    p.freq = r->freq, p.scale = (float)r->scale;
    p.sign = (flags & TG_FLAG_ROPE_INVERSE) ? -1.f : 1.f;
    p.tokens = tokens, p.positions = positions;
    return rope_run<T, false>(p, r->layout, static_cast<cudaStream_t>(stream), op);
}

template <typename T>
int append(const tg_kv_append_args* a, tg_stream_t stream, const char* op) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_cache(a->cache, op);
    if (rc == TG_OK) rc = check_table(a->pages, a->cache, a->tokens, a->q_indptr, a->seq_len, op);
    if (rc == TG_OK && a->rope) rc = check_rope(a->rope, a->cache->dim, op);
    if (rc == TG_OK && a->rope) rc = check_rot(a->rope, op);
    if (rc != TG_OK) return rc;
    if (a->flags & ~TG_FLAG_BOUNDS_CHECK) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if (a->q && (!a->q_out || a->q_heads < 0)) return set_error(TG_EINVAL, "%s: q without q_out, or q_heads < 0", op);
    if (a->tokens == 0) return TG_OK;
    if (!a->k.data || !a->v.data) return set_error(TG_EINVAL, "%s: null k/v", op);
    const bool with_q = a->q && a->q_heads > 0;
    if (with_q && (!a->q->data || !a->q_out->data)) return set_error(TG_EINVAL, "%s: null q/q_out", op);
    const tg_paged_kv& c = *a->cache;
    const tg_csr& t = *a->pages;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->flags & TG_FLAG_BOUNDS_CHECK) {
        rc = paged_bounds_check(t, c.page_size, a->seq_len, INT64_MAX, a->tokens, a->q_indptr, INT64_MAX, nullptr, 0,
                                true, op, st);
        if (rc != TG_OK) return rc;
    }
    RopeParams<T> p = {};
    p.k = static_cast<const T*>(a->k.data), p.ko = static_cast<T*>(c.k);
    p.v = static_cast<const T*>(a->v.data), p.vo = static_cast<T*>(c.v);
    p.k_tok = a->k.token_stride, p.k_head = a->k.head_stride;
    p.v_tok = a->v.token_stride, p.v_head = a->v.head_stride;
    p.ko_page = c.k_page_stride, p.ko_slot = c.k_slot_stride, p.ko_head = c.k_head_stride;
    p.vo_page = c.v_page_stride, p.vo_slot = c.v_slot_stride, p.vo_head = c.v_head_stride;
    p.kv_rows = c.heads, p.dim = c.dim;
    if (with_q) {
        p.q = static_cast<const T*>(a->q->data), p.qo = static_cast<T*>(a->q_out->data);
        p.q_tok = a->q->token_stride, p.q_head = a->q->head_stride;
        p.qo_tok = a->q_out->token_stride, p.qo_head = a->q_out->head_stride;
        p.q_rows = a->q_heads;
    }
    if (a->rope) {
        p.rot = a->rope->rot_dim, p.freq = a->rope->freq, p.scale = (float)a->rope->scale;
    }
    p.sign = 1.f;
    p.tokens = a->tokens, p.positions = a->positions, p.position_base = a->position_base;
    p.q_indptr = a->q_indptr, p.seq_len = a->seq_len, p.indptr = t.indptr, p.indices = t.indices;
    p.rows = t.rows, p.pages = c.pages, p.nnz = t.nnz, p.page_size = c.page_size;
    return rope_run<T, true>(p, a->rope ? a->rope->layout : TG_ROPE_HALF, st, op);
}

}  // namespace
}  // namespace tg

extern "C" {

#define TG_ROPE_ENTRY(SUFFIX, T)                                                                                     \
    int tg_rope_##SUFFIX(const tg_rope* r, const tg_rows* x, const tg_rows* y, int64_t tokens, int32_t heads,        \
                         int32_t dim, const int64_t* positions, uint32_t flags, tg_stream_t stream) {                \
        return tg::rope<T>(r, x, y, tokens, heads, dim, positions, flags, stream, "tg_rope_" #SUFFIX);               \
    }                                                                                                                \
    int tg_kv_append_##SUFFIX(const tg_kv_append_args* a, tg_stream_t stream) {                                      \
        return tg::append<T>(a, stream, "tg_kv_append_" #SUFFIX);                                                    \
    }
TG_ROPE_ENTRY(f32, float)
TG_ROPE_ENTRY(f16, __half)
TG_ROPE_ENTRY(bf16, __nv_bfloat16)

}  // extern "C"
