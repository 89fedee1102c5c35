// Rotary positions and the paged-cache append (tg_rope_*, tg_kv_append_*).
//
// Pair i of a head's rotating elements (a, b) becomes scale * (a cos t - b sin t,
// b cos t + a sin t) with t = position * freq[i]; the gradient is the same with -t.  One
// kernel serves both calls: its rows are the heads of a token, of three kinds -- q (rotated
// into an output), k (rotated into the token's cache slot) and v (copied there).
//
// * Bound: HBM.  Each element is read once and written once, 16 bytes a load, and the
//   angles cost no traffic: a CTA takes a few tokens, computes their cosines and sines once
//   into shared memory, and all heads of these tokens use them.  16383 tokens of 32 heads of 128
//   in bfloat16 (268 MB): 47-49 us, 5.6 TB/s; an append of 572 MB: 98-101 us, 5.8 TB/s (the
//   measured copy: 6.5 TB/s).
// * The angle and its rest after whole turns (2 pi in two parts, after Cody and Waite) are
//   64-bit, so a position of 1e6 is as exact as position 1; the sine and cosine of the rest,
//   their product with the scale, the rotation itself and its sum are 32-bit, rounded once to the
//   output's type (for float32 outputs 3.5e-8 off on average, where a 64-bit sine gives 2.9e-8).
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
    int lanes, chunks, blocks;  // threads along a row, items of a row, rounds of the threads over them
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
        if constexpr (VEC > 1 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 x = unpack2<T>(reinterpret_cast<const uint32_t*>(v)[i / 2]);
                f[i] = x.x, f[i + 1] = x.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = to_f32(v[i]);
        }
    }
    __device__ __forceinline__ void put(const float (&f)[VEC]) {
        if constexpr (VEC > 1 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) reinterpret_cast<uint32_t*>(v)[i / 2] = pack2<T>(f[i], f[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(f[i]);
        }
    }
};

constexpr int kRopeThreads = 256;
constexpr int kRopeTile = 32;         // most tokens of a CTA
constexpr int kRopeSmem = 32 * 1024;  // most bytes of cosines and sines of a CTA

// VEC elements (a pack) are moved at once: 16 bytes where rows, strides and the parts of a row are
// multiples of that, else single elements.  A thread's item is two packs of a row: the two halves
// of its pairs (HALF, or single elements of neighbouring pairs), or two packs of whole pairs or
// copied elements, a stretch of a row apart so that the threads' packs lie side by side.  The
// first item's packs are under way while the sines are made.
template <typename T, int VEC, bool HALF, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads, APPEND ? 6 : 5) rope_kernel(const RopeParams<T> p) {
    extern __shared__ float4 s_turn4[];  // scale * (cos, sin) of [tile][pairs], two pairs in one float4
    float2* const s_turn = reinterpret_cast<float2*>(s_turn4);
    __shared__ double s_pos[kRopeTile];
    __shared__ int64_t s_page[kRopeTile];  // the token's cache page, -1: no such slot
    __shared__ int64_t s_slot[kRopeTile];
    using P = Pack<T, VEC>;
    constexpr bool kApart = HALF || VEC == 1;  // a pair's elements are in different packs
    // The next packs under way cost 10 registers, a CTA on an SM: worth it for the rotation alone
    // (47 against 54 us for 268 MB), not for the append (106 against 98 us for 572 MB), which waits for
    // page numbers too.
    constexpr bool kAhead = !APPEND;
    constexpr int kPairs = kApart ? VEC : VEC / 2;  // of an item's pack
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

    const int pairs = p.rot / 2, packs = p.dim / VEC;
    const int turning = kApart ? pairs / VEC : p.rot / VEC;  // packs (or pairs of packs) that turn
    const int rows = (p.q_rows + (APPEND ? 2 * p.kv_rows : 0)) * p.blocks, step = blockDim.x / p.lanes;
    struct Item {
        P a, b;
        T* out;
        int ia, ib;  // places of the packs; ib < 0: none
        int tt;      // token of the tile, -1: nothing turns
    };
    int tt = 0, row = tid / p.lanes - step;
    auto next = [&](Item& x) {  // the thread's next item, its loads under way
        for (;;) {
            row += step;
            while (row >= rows) {
                row -= rows;
                ++tt;
            }
            if (tt >= tile) return false;
            const int r = p.blocks == 1 ? row : row / p.blocks;
            const int c = tid % p.lanes + (p.blocks == 1 ? 0 : (row - r * p.blocks) * p.lanes);
            if (c >= p.chunks) continue;
            const int64_t t = t0 + tt;
            const T* in;
            bool turns = true;
            if (!APPEND || r < p.q_rows) {
                in = p.q + t * p.q_tok + r * p.q_head;
                x.out = p.qo + t * p.qo_tok + r * p.qo_head;
            } else {
                const int64_t page = s_page[tt];
                if (page < 0) continue;
                const int h = r - p.q_rows;
                turns = h < p.kv_rows;
                if (turns) {
                    in = p.k + t * p.k_tok + h * p.k_head;
                    x.out = p.ko + page * p.ko_page + s_slot[tt] * p.ko_slot + h * p.ko_head;
                } else {
                    in = p.v + t * p.v_tok + (h - p.kv_rows) * p.v_head;
                    x.out = p.vo + page * p.vo_page + s_slot[tt] * p.vo_slot + (h - p.kv_rows) * p.vo_head;
                }
            }
            x.tt = turns ? tt : -1;
            if (kApart && turns) {
                if (c < turning) {
                    x.ia = HALF ? c : 2 * c;
                    x.ib = HALF ? turning + c : 2 * c + 1;
                } else {  // copied, behind the turning ones
                    const int rest = p.chunks - turning;
                    x.ia = turning + c;
                    x.ib = x.ia + rest < packs ? x.ia + rest : -1;
                    x.tt = -1;
                }
            } else {
                x.ia = c;
                x.ib = c + p.chunks < packs ? c + p.chunks : -1;
            }
            x.a = reinterpret_cast<const P*>(in)[x.ia];
            if (x.ib >= 0) x.b = reinterpret_cast<const P*>(in)[x.ib];
            return true;
        }
    };
    // The sines of pair j of pack c of a token: float4 j / 2 of all packs side by side, so that lanes
    // read them without bank conflicts.
    auto place = [&](int c, int j) { return kPairs == 1 ? c : ((j >> 1) * turning + c) * 2 + (j & 1); };
    auto sines = [&](const float2* turn, int c, float2* cs) {
        if constexpr (kPairs == 1) {
            cs[0] = turn[c];
        } else {
#pragma unroll
            for (int j = 0; j < kPairs; j += 2) {
                const float4 v = *reinterpret_cast<const float4*>(turn + place(c, j));
                cs[j] = make_float2(v.x, v.y);
                cs[j + 1] = make_float2(v.z, v.w);
            }
        }
    };
    auto turn_pack = [&](P& v, int i, const float2* turn) {  // whole pairs
        if (i >= turning) return;
        float2 cs[kPairs];
        float f[VEC];
        sines(turn, i, cs);
        v.get(f);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            const float u = f[2 * j], w = f[2 * j + 1];
            f[2 * j] = u * cs[j].x - w * cs[j].y;
            f[2 * j + 1] = w * cs[j].x + u * cs[j].y;
        }
        v.put(f);
    };
    Item x;
    bool have = next(x);

    for (int i = tid; i < tile * pairs; i += blockDim.x) {
        const int k = i / pairs;
        const double t = s_pos[k] * p.freq[i - k * pairs];
        const double whole = rint(t * 0.15915494309189533577);  // turns
        const double rest = fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, t));  // 2 pi in two parts
        float s, c;
        sincospif((float)(rest * 0.31830988618379067154), &s, &c);
        const int pair = i - k * pairs;
        s_turn[k * pairs + place(pair / kPairs, pair % kPairs)] = make_float2(c * p.scale, s * p.scale * p.sign);
    }
    __syncthreads();

    while (have) {
        Item y;
        if constexpr (kAhead) have = next(y);
        if (x.tt >= 0) {
            const float2* turn = s_turn + x.tt * pairs;
            if constexpr (kApart) {
                float2 cs[kPairs];
                sines(turn, HALF ? x.ia : x.ia / 2, cs);
                float f[VEC], g[VEC];
                x.a.get(f);
                x.b.get(g);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = f[j], w = g[j];
                    f[j] = u * cs[j].x - w * cs[j].y;
                    g[j] = w * cs[j].x + u * cs[j].y;
                }
                x.a.put(f);
                x.b.put(g);
            } else {
                turn_pack(x.a, x.ia, turn);
                if (x.ib >= 0) turn_pack(x.b, x.ib, turn);
            }
        }
        reinterpret_cast<P*>(x.out)[x.ia] = x.a;
        if (x.ib >= 0) reinterpret_cast<P*>(x.out)[x.ib] = x.b;
        if constexpr (kAhead) x = y;
        else have = next(x);
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
    const bool half = layout == TG_ROPE_HALF;
    const bool wide = all % 16 == 0 && p.dim % WIDE == 0 && p.rot % (half ? 2 * WIDE : WIDE) == 0;
    const int vec = wide ? WIDE : 1;
    p.chunks = half || !wide ? p.rot / 2 / vec + ((p.dim - p.rot) / vec + 1) / 2 : (p.dim / vec + 1) / 2;
    p.lanes = std::min(p.chunks, kRopeThreads);
    p.blocks = (p.chunks + p.lanes - 1) / p.lanes;
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
    p.q_tok = stride_of(tokens, x->token_stride), p.q_head = stride_of(heads, x->head_stride);
    p.qo_tok = stride_of(tokens, y->token_stride), p.qo_head = stride_of(heads, y->head_stride);
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
    p.k_tok = stride_of(a->tokens, a->k.token_stride), p.k_head = stride_of(c.heads, a->k.head_stride);
    p.v_tok = stride_of(a->tokens, a->v.token_stride), p.v_head = stride_of(c.heads, a->v.head_stride);
    p.ko_page = stride_of(c.pages, c.k_page_stride), p.vo_page = stride_of(c.pages, c.v_page_stride);
    p.ko_slot = stride_of(c.page_size, c.k_slot_stride), p.vo_slot = stride_of(c.page_size, c.v_slot_stride);
    p.ko_head = stride_of(c.heads, c.k_head_stride), p.vo_head = stride_of(c.heads, c.v_head_stride);
    p.kv_rows = c.heads, p.dim = c.dim;
    if (with_q) {
        p.q = static_cast<const T*>(a->q->data), p.qo = static_cast<T*>(a->q_out->data);
        p.q_tok = stride_of(a->tokens, a->q->token_stride), p.q_head = stride_of(a->q_heads, a->q->head_stride);
        p.qo_tok = stride_of(a->tokens, a->q_out->token_stride), p.qo_head = stride_of(a->q_heads, a->q_out->head_stride);
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
