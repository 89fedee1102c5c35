// Pieces of the kernels that rotate rows (tg_rope.cu, tg_norm_rope.cu): packs of a row, the angle of a
// pair, the cache slot of a new token.
#pragma once

#include "tg_paged.cuh"

namespace tg {

constexpr int kRopeThreads = 256;
constexpr int kRopeTile = 32;         // most tokens of a CTA
constexpr int kRopeSmem = 32 * 1024;  // most bytes of cosines and sines of a CTA

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

// The tokens of a call; but for tokens and positions, of an append only.
struct NewTokens {
    int64_t tokens;
    const int64_t* positions;
    int64_t position_base;
    const int64_t *q_indptr, *seq_len, *indptr, *indices;
    int64_t rows, pages, nnz, page_size;
};

// The place of token t in its sequence, and the cache page (-1: no such slot) and slot of that place.
__device__ __forceinline__ int64_t slot_of_token(const NewTokens& p, int64_t t, int64_t& page, int64_t& slot) {
    const int64_t b = sequence_of(p.q_indptr, p.rows, t);
    int64_t first, n, page0, npages;
    tokens_of(p.q_indptr, p.tokens, b, first, n);
    pages_of(p.indptr, p.nnz, b, page0, npages);
    const int64_t at = p.seq_len[b] - n + (t - first);
    int64_t found = -1;
    if (at >= 0 && t >= first && t < first + n) {
        const int64_t j = at / p.page_size;
        if (j < npages) found = p.indices[page0 + j];
        if (found >= p.pages) found = -1;
        slot = at - j * p.page_size;
    }
    page = found;
    return at;
}

// scale * (cos, sign * sin) of position * freq.  The angle and its rest after whole turns (2 pi in two
// parts, after Cody and Waite) are 64-bit.  QUICK: sine and cosine of the rest by the special-function
// unit, 2^-21 off (absolute), a quarter of the instructions: for outputs of 16 bits.
template <bool QUICK = false>
__device__ __forceinline__ float2 turn_of(double position, double freq, float scale, float sign) {
    const double t = position * freq;
    const double whole = rint(t * 0.15915494309189533577);  // turns
    const double rest = fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, t));  // 2 pi in two parts
    float s, c;
    if constexpr (QUICK) __sincosf((float)rest, &s, &c);
    else sincospif((float)(rest * 0.31830988618379067154), &s, &c);
    return make_float2(c * scale, s * scale * sign);
}

constexpr int kMaxRot = 2 * (kRopeSmem / 8);  // one token's cosines and sines fit a CTA

inline int check_rot(const tg_rope* r, const char* op) {
    return r->rot_dim > kMaxRot ? set_error(TG_EUNSUPPORTED, "%s: rot_dim above %d", op, kMaxRot) : TG_OK;
}

// The checks of an append; done: nothing is left to do (tg_paged_host.cu).
int check_append(const tg_kv_append_args* a, const char* op, cudaStream_t st, bool& done);

// The tokens of a checked append.
inline void new_tokens(const tg_kv_append_args& a, NewTokens& p) {
    p.tokens = a.tokens, p.positions = a.positions, p.position_base = a.position_base;
    p.q_indptr = a.q_indptr, p.seq_len = a.seq_len, p.indptr = a.pages->indptr, p.indices = a.pages->indices;
    p.rows = a.pages->rows, p.pages = a.cache->pages, p.nnz = a.pages->nnz, p.page_size = a.cache->page_size;
}

}  // namespace tg
