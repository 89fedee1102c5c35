// Parameters and device pieces shared by the shared-prefix attention kernels.
//
// The keys of a sequence are cut into parts: splits of the shared prefix and chunks of the
// sequence's own pages.  Each part leaves, for each of its rows (token, query head), the
// maximum m and sum l of exp2(s - m) over its keys (s: the scores times log2 e) and the
// sum of exp2(s - m) v, all in 32 bits; the parts of a row are joined by
//   M = max m_i,  out = sum_i exp2(m_i - M) o_i / sum_i exp2(m_i - M) l_i.
#pragma once

#include <cuda.h>

#include "tg_paged.cuh"

namespace tg {

struct AttnParams {
    const void *q, *k, *v;
    void* out;
    float* lse;
    int64_t q_tok, q_head, o_tok, o_head;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int pages, page_size, page_shift;  // page_shift: log2(page_size), -1 where it is no power of two
    int q_heads, kv_heads, group;
    int tokens, rows;  // queries, sequences
    const int64_t *q_indptr, *indptr, *indices, *seq_len, *prefix_pages;
    int64_t nnz;
    int max_seq, max_q, prefix_len;
    float scale_log2;
    int causal;
    // parts
    int prefix_splits, prefix_chunk;  // most parts of a row over the prefix; keys of a split
    // the tcgen05 kernel over the prefix: its CTAs share prefix_work steps of 128 keys evenly,
    // prefix_steps for each (head, row tile) in turn, prefix_tiles row tiles
    int prefix_work, prefix_per_unit, prefix_ctas, prefix_steps, prefix_tiles;  // prefix_ctas 0: splits of prefix_chunk keys
    int own_chunks, own_chunk;        // most chunks of a sequence, keys of a chunk
    int own_pieces;                   // the tcgen05 kernel: (head, chunk, sequence, row tile)
    int tiles;                        // row tiles of a sequence (own) or of all rows (prefix)
    int over_prefix;                  // the tcgen05 kernel: the prefix, else the sequences' own pages
    int prefix_units;                 // the kernel for few rows: its first blocks go over the prefix
    int fill;                         // the only part, of own pages, tokens by q_indptr: fill_unanswered
    int direct;                       // the only part: rows are finished here
    float* part_o;                    // [part][token][head][dim]
    float2* part_ml;                  // [part][token][head]: m, l
};

// One sequence as the kernels see it: its tokens, how many of them are answered (the first max_q),
// its own pages and length.
struct Sequence {
    int64_t page0;
    int first, n, asked, len;
};

__device__ __forceinline__ Sequence sequence(const AttnParams& p, int64_t b) {
    Sequence s;
    int64_t first, n, npages;
    tokens_of(p.q_indptr, p.tokens, b, first, n);
    pages_of(p.indptr, p.nnz, b, s.page0, npages);
    s.first = (int)first;
    s.n = (int)n;
    s.asked = min(s.n, p.max_q);
    const int64_t len = min(min(p.seq_len[b], npages * p.page_size), (int64_t)p.max_seq);
    s.len = (int)max(len, (int64_t)0);
    return s;
}

// Keys that the i-th query of a sequence sees among the first `whole`, of `total` keys.
__device__ __forceinline__ int keys_seen(const AttnParams& p, const Sequence& s, int i, int64_t total, int whole) {
    if (!p.causal) return whole;
    return (int)min(max(total - s.n + i + 1, (int64_t)0), (int64_t)whole);
}

// Keys of the prefix (`whole` keys) that token t of sequence s sees: none where s does not answer it.
__device__ __forceinline__ int prefix_seen(const AttnParams& p, const Sequence& s, int t, int whole) {
    const int i = t - s.first;
    return i < 0 || i >= s.asked ? 0 : keys_seen(p, s, i, (int64_t)whole + s.len, whole);
}

// A call without a join: the rows of tokens that no sequence answers (past its first max_q, before
// the first sequence or after the last one) are no CTA's of the kernel over the own pages, so warp
// `warp` of `warps` writes its share of them at its end, zeros and -inf: one sequence after the
// other, and all warps share the tokens of none.  Instances of their own have it: calls with a join
// took 53 us for 50 and 60 for 55 with this code in the kernel, run or not, and a launch of its own
// costs small calls 2 to 4 of 21 to 24 us.
template <typename T, int D>
__device__ __forceinline__ void fill_unanswered(const AttnParams& p, int64_t warp, int64_t warps) {
    const int lane = threadIdx.x & 31;
    auto fill = [&](int64_t t0, int64_t t1, int64_t mine, int64_t all) {
        for (int64_t t = t0 + mine; t < t1; t += all)
            for (int h = 0; h < p.q_heads; ++h) {
                if (lane < D / 8)
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.o_tok + h * p.o_head + lane * 8) = make_uint4(0, 0, 0, 0);
                if (p.lse && lane == 0) p.lse[t * p.q_heads + h] = -INFINITY;
            }
    };
    const int64_t all = p.tokens, begin = min(max(p.q_indptr[0], (int64_t)0), all), end = max(min(p.q_indptr[p.rows], all), begin);
    fill(0, begin, warp, warps);
    fill(end, all, warp, warps);
    for (int64_t b = warp; b < p.rows; b += warps) {
        int64_t first, n;
        tokens_of(p.q_indptr, p.tokens, b, first, n);
        if (n > p.max_q) fill(first + p.max_q, first + n, 0, 1);
    }
}

// The first step of part i of n near-even shares of `all` steps (the first all % n have one more),
// and the share that has step x.
__host__ __device__ __forceinline__ int share_start(int all, int n, int i) {
    const int q = all / n, more = all - q * n;
    return i * q + (i < more ? i : more);
}
__host__ __device__ __forceinline__ int share_of(int all, int n, int x) {
    const int q = all / n, more = all - q * n;
    return x < more * (q + 1) ? x / (q + 1) : more + (x - more * (q + 1)) / q;
}
// The same for the CTAs over the prefix: prefix_per_unit of them for each (head, row tile), or even
// shares of all steps where that is 0.
__host__ __device__ __forceinline__ int prefix_start(const AttnParams& p, int cta) {
    if (!p.prefix_per_unit) return share_start(p.prefix_work, p.prefix_ctas, cta);
    const int u = cta / p.prefix_per_unit;
    return u * p.prefix_steps + share_start(p.prefix_steps, p.prefix_per_unit, cta - u * p.prefix_per_unit);
}
__host__ __device__ __forceinline__ int prefix_cta(const AttnParams& p, int x) {
    if (!p.prefix_per_unit) return share_of(p.prefix_work, p.prefix_ctas, x);
    const int u = x / p.prefix_steps;
    return u * p.prefix_per_unit + share_of(p.prefix_steps, p.prefix_per_unit, x - u * p.prefix_steps);
}

// Page and slot of token `at` of a page list; page -1 where the list names no page of the cache.
__device__ __forceinline__ void locate(const AttnParams& p, const int64_t* list, int at, int& page, int& slot) {
    int j;
    if (p.page_shift >= 0) {
        j = at >> p.page_shift;
        slot = at & (p.page_size - 1);
    } else {
        j = at / p.page_size;
        slot = at - j * p.page_size;
    }
    const int64_t id = __ldg(list + j);
    page = id >= 0 && id < p.pages ? (int)id : -1;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The value that P is taken relative to, for a row's maximum `top`.  float16 has no number below
// 2^-24: beside a largest weight of 1, thousands of weights of 2^-26 would all round to nothing.
// LIFT (15 or less) puts the largest weight at 2^LIFT instead.  Maxima of 2^20 and above, where top -
// LIFT would be rounded, stay as they are.
template <typename T, int LIFT>
__device__ __forceinline__ float reference(float top) {
    if constexpr (std::is_same<T, __half>::value) return fabsf(top) < 1048576.f ? top - (float)LIFT : top;
    else return top;
}
// Whether one of the eight 16-bit numbers in v is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint4 v) {
    constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    bool bad = false;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & kExp) == kExp || ((w[i] >> 16) & kExp) == kExp;
    return bad;
}

// A box of a [page][head][slot][dim] map: 64 elements from x of the rows from `slot`.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                         uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        "\n\t}" ::"r"(dst),
        "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}

// Tensor maps of the keys and values as [page][head][slot][dim], boxes of box_rows slots of 64
// elements of one head, rows of 128 bytes swizzled by 128 bytes (tg_paged_host.cu).
int cache_maps(const AttnParams& p, bool is_half, int dim, int box_rows, CUtensorMap* k, CUtensorMap* v);

// tg_prefix_attn_tc.cu
template <typename T>
int attn_tc_run(const AttnParams& p, int dim, int ctas, bool pdl, cudaStream_t st);

}  // namespace tg
