// Attention of a batch that shares a prefix (tg_prefix_attention_*): the kernel for few
// rows, the join of the parts, planning and the C entry points.
#include <algorithm>
#include <numeric>

#include "tg_prefix_attn.cuh"

namespace tg {
namespace {

// ------------------------------------------------------------------ matrix instructions
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// ------------------------------------------------------------------ few rows
// One warp: RT*16 rows (of one sequence's tokens x group, or of all tokens over the prefix), one
// key head, one chunk of keys, 16 at a time.
//
// Bound: HBM (the keys and values of a chunk are read once for 16 RT rows).  16 keys are a TMA box
// of 64 columns (or as many boxes as pages cut them into), which lands swizzled, free of bank
// conflicts for ldmatrix; nothing synchronises warps, so an SM holds as many as its shared memory
// does, at different places of their chunks, and the chain of page table, page and result is
// hidden.  The rows are the 16 rows of mma.m16n8k16; S stays in registers and is the A operand of
// the second product as it lies.  64 sequences of 4096 keys, 8 heads of 128, one query each: 1.07 GB
// in 179 us, 6.0 TB/s, 92 % of the measured copy (four warps a CTA with 16-byte copies: 4.1 TB/s).
constexpr int kStepKeys = 16;

template <int D, int RT>
struct RowCfg {
    static constexpr int kHalves = (D + 63) / 64;
    static constexpr int kBox = kStepKeys * 128;  // bytes of 64 columns of 16 rows
    static constexpr int kStage = 2 * kHalves * kBox;  // K then V
    static constexpr int kStages = 3;
    static constexpr int kPitch = D * 2 + 16;  // of the queries, padded
    static constexpr int kQ = RT == 1 ? 0 : RT * 16 * kPitch;
    static constexpr int kSmem = kStages * kStage + kQ + 64;  // and the barriers
    static_assert(RT * 16 * kStepKeys * 4 <= kHalves * kBox, "a step's P fits its K tile");
};

template <typename T, int D, int RT, bool FILL>
__global__ void __launch_bounds__(32) attn_rows_kernel(const AttnParams p, const int box,
                                                       const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap) {
    using C = RowCfg<D, RT>;
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    constexpr int S = C::kStages;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* const sq = smem + S * C::kStage;
    uint64_t* const bar = reinterpret_cast<uint64_t*>(sq + C::kQ);
    const int lane = threadIdx.x;
    pdl_trigger();
    // The grids of a call complete in order: this one (the second) ends after the first.
    struct AtEnd {
        const AttnParams& p;
        __device__ ~AtEnd() {
            if constexpr (FILL)
                fill_unanswered<T, D>(p, (int64_t)blockIdx.y * gridDim.x + blockIdx.x, (int64_t)gridDim.y * gridDim.x);
            if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
        }
    } at_end{p};

    // ---- which rows, which keys
    const int h = blockIdx.y;
    const bool over_prefix = blockIdx.x < p.prefix_units;
    Sequence s;
    const int64_t* list;
    int tile, part, keys, k0, k1;
    if (over_prefix) {
        part = blockIdx.x % p.prefix_splits;
        tile = blockIdx.x / p.prefix_splits;
        s.first = 0;
        s.n = s.asked = p.tokens;
        list = p.prefix_pages;
        keys = p.prefix_len;
        k0 = part * p.prefix_chunk;
        k1 = min(keys, k0 + p.prefix_chunk);
    } else {
        const int x = blockIdx.x - p.prefix_units, c = x % p.own_chunks, u = x / p.own_chunks;
        tile = u % p.tiles;
        s = sequence(p, u / p.tiles);
        list = p.indices + s.page0;
        keys = s.len;
        k0 = c * p.own_chunk;
        k1 = min(keys, k0 + p.own_chunk);
        part = p.prefix_splits + c;
        if (k0 >= keys && !p.direct) return;  // no such chunk: the join does not ask for it
    }
    const int row0 = tile * RT * 16, nrows = min(s.asked * p.group - row0, RT * 16);
    if (nrows <= 0) return;
    if (!over_prefix)  // no row sees more than the last one
        k1 = min(k1, keys_seen(p, s, (row0 + nrows - 1) / p.group, keys, keys));
    const int steps = max(0, (k1 - k0 + kStepKeys - 1) / kStepKeys);

    if (lane == 0) {
        for (int i = 0; i < S; ++i) mbar_init(&bar[i], 1);
        fence_mbar_init();
    }
    __syncwarp();
    const uint32_t ring = smem_addr(smem);
    const int boxes = kStepKeys / box;
    // Lane l: the page of box l of a step, -1 past the end.  A page that does not exist is fetched
    // from behind the last one, which reads as zeros.
    auto find = [&](int i, int& page, int& slot) {
        const int at = k0 + i * kStepKeys + lane * box;
        page = -1;
        slot = 0;
        if (lane < boxes && at < k1) {
            locate(p, list, at, page, slot);
            if (page < 0) page = p.pages;
        }
    };
    auto fetch = [&](int stage, int page, int slot) {
        const uint32_t dst = ring + stage * C::kStage, there = __ballot_sync(kFull, page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&bar[stage], __popc(there) * box * C::kHalves * 256);
        __syncwarp();
        for (int i = 0; i < boxes; ++i) {
            const int pg = __shfl_sync(kFull, page, i), sl = __shfl_sync(kFull, slot, i);
            if (!(there >> i & 1)) continue;
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half) {
                load_box(dst + half * C::kBox + i * box * 128, &kmap, half * 64, sl, h, pg, smem_addr(&bar[stage]));
                load_box(dst + (C::kHalves + half) * C::kBox + i * box * 128, &vmap, half * 64, sl, h, pg, smem_addr(&bar[stage]));
            }
        }
    };
    // A 16-byte chunk of a row of a tile; rows of 128 bytes, chunks swizzled by the row.
    auto chunk_at = [&](uint32_t tile_at, int r, int c) { return tile_at + (c >> 3) * C::kBox + r * 128 + (((c ^ r) & 7) << 4); };
    {
        int page[S], slot[S];
#pragma unroll
        for (int i = 0; i < S; ++i) find(i, page[i], slot[i]);
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i < steps) fetch(i, page[i], slot[i]);
    }

    // ---- queries: fragments in registers for one row tile, in shared memory for two; zeros for
    // rows that are not there
    uint32_t qf[RT == 1 ? D / 16 : 1][4];
    const uint32_t qaddr = smem_addr(sq) + (lane & 15) * C::kPitch + (lane >> 4) * 16;
    const char* qbase = static_cast<const char*>(p.q) + (int64_t)h * p.group * p.q_head * 2;
    if constexpr (RT == 1) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = (lane >> 2) + 8 * e, f = row0 + (r < nrows ? r : 0);
            const char* q = qbase + ((int64_t)(s.first + f / p.group) * p.q_tok + f % p.group * p.q_head + 2 * (lane & 3)) * 2;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    qf[kk][2 * x + e] = r < nrows ? __ldg(reinterpret_cast<const uint32_t*>(q + kk * 32 + x * 16)) : 0;
        }
    } else {
#pragma unroll 4
        for (int i = lane; i < RT * 16 * CH; i += 32) {
            const int r = i / CH, c = i % CH, f = row0 + (r < nrows ? r : 0);
            uint4 v = __ldg(reinterpret_cast<const uint4*>(
                qbase + ((int64_t)(s.first + f / p.group) * p.q_tok + f % p.group * p.q_head) * 2 + c * 16));
            if (r >= nrows) v = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(sq + r * C::kPitch + c * 16) = v;
        }
        __syncwarp();
    }
    // ---- keys that each of the thread's rows sees (none where there is no row)
    int seen[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = rt * 16 + (lane >> 2) + 8 * e;
            seen[rt][e] = 0;
            if (r < nrows) {
                const int i = (row0 + r) / p.group;
                if (!over_prefix) {
                    seen[rt][e] = keys_seen(p, s, i, keys, keys);
                } else if (!p.causal && !p.q_indptr) {
                    seen[rt][e] = keys;
                } else {
                    seen[rt][e] = prefix_seen(p, sequence(p, sequence_of(p.q_indptr, p.rows, i)), i, keys);
                }
            }
        }

    float o[RT][D / 8][4], m[RT][2], l[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt][0] = m[rt][1] = -INFINITY;
        l[rt][0] = l[rt][1] = 0.f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rt][n][e] = 0.f;
    }

    int stage = 0, phase = 0;
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
        int page, slot;
        find(it + S, page, slot);
        if (!__all_sync(kFull, mbar_wait(&bar[stage], phase))) {
            ok = false;
            break;
        }
        const uint32_t kt = ring + stage * C::kStage, vt = kt + C::kHalves * C::kBox;
        const int key0 = k0 + it * kStepKeys, step_end = min(key0 + kStepKeys, k1);
        // Values past the end are zeros: a box may hold anything there, and 0 * NaN is not 0 (it is
        // the last step, so no later box lands on what is written here).
        if (key0 + kStepKeys > k1) {
            for (int i = (k1 - key0) * 8 + lane; i < kStepKeys * 8; i += 32)
#pragma unroll
                for (int half = 0; half < C::kHalves; ++half)
                    *reinterpret_cast<uint4*>(smem + (vt - ring) + half * C::kBox + i * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }

        float sc[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[rt][n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t b[4];
            ldmatrix4(chunk_at(kt, (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)), b);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if constexpr (RT == 1) {
                    mma16816<T>(sc[rt][0], qf[kk], b[0], b[1]);
                    mma16816<T>(sc[rt][1], qf[kk], b[2], b[3]);
                } else {
                    uint32_t a[4];
                    ldmatrix4(qaddr + rt * 16 * C::kPitch + kk * 32, a);
                    mma16816<T>(sc[rt][0], a, b[0], b[1]);
                    mma16816<T>(sc[rt][1], a, b[2], b[3]);
                }
            }
        }

        uint32_t pf[RT][4];
        bool part_seen = false;  // a row of this lane sees only some of the step's keys
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = rt * 16 + (lane >> 2) + 8 * e;
                part_seen |= r < nrows && seen[rt][e] < step_end;
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float& v = sc[rt][n][2 * e + x];
                        v = key0 + n * 8 + 2 * (lane & 3) + x < seen[rt][e] ? v * p.scale_log2 : -INFINITY;
                        mx = fmaxf(mx, v);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
                const float mn = fmaxf(m[rt][e], reference<T, 15>(mx)), base = mn == -INFINITY ? 0.f : mn;
                const float keep = exp2_fast(m[rt][e] - base);
                m[rt][e] = mn;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float& v = sc[rt][n][2 * e + x];
                        v = exp2_fast(v - base);
                        sum += v;
                    }
                l[rt][e] = l[rt][e] * keep + sum;
                if (__any_sync(kFull, keep != 1.f)) {
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[rt][n][2 * e] *= keep;
                        o[rt][n][2 * e + 1] *= keep;
                    }
                }
                // P is rounded to the values' type for the product, as the output is: relative
                // errors of half an ulp that average out over the keys (in float16, weights below
                // 2^-40 of a part's largest are lost).  l sums the unrounded P.
                pf[rt][e] = pack2<T>(sc[rt][0][2 * e], sc[rt][0][2 * e + 1]);
                pf[rt][2 + e] = pack2<T>(sc[rt][1][2 * e], sc[rt][1][2 * e + 1]);
            }

        // A value that only some rows see must not reach the others through 0 * NaN: where a
        // step is seen in part and holds an infinity or NaN, its product is taken row by row.
        bool by_rows = false;
        if (__any_sync(kFull, part_seen)) {
            bool bad = false;
            for (int i = lane; i < kStepKeys * CH; i += 32)
                bad |= any_nonfinite<T>(*reinterpret_cast<const uint4*>(smem + (chunk_at(vt, i / CH, i % CH) - ring)));
            by_rows = __any_sync(kFull, bad);
        }
        if (by_rows) {
            __syncwarp();
            float* sp = reinterpret_cast<float*>(smem + (kt - ring));  // the K tile is done with
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sp[(rt * 16 + (lane >> 2) + 8 * (e >> 1)) * kStepKeys + n * 8 + 2 * (lane & 3) + (e & 1)] = sc[rt][n][e];
            __syncwarp();
#pragma unroll 1
            for (int key = 0; key < kStepKeys; ++key) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (key0 + key >= seen[rt][e]) continue;
                        const float w = sp[(rt * 16 + (lane >> 2) + 8 * e) * kStepKeys + key];
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) {
                            const T* vr = reinterpret_cast<const T*>(smem + (chunk_at(vt, key, n) - ring)) + 2 * (lane & 3);
                            o[rt][n][2 * e] += w * to_f32(vr[0]);
                            o[rt][n][2 * e + 1] += w * to_f32(vr[1]);
                        }
                    }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a box will land where P is
        } else {
#pragma unroll
            for (int dn = 0; dn < D / 16; ++dn) {
                uint32_t b[4];
                ldmatrix4_trans(chunk_at(vt, lane & 15, dn * 2 + (lane >> 4)), b);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    mma16816<T>(o[rt][2 * dn], pf[rt], b[0], b[1]);
                    mma16816<T>(o[rt][2 * dn + 1], pf[rt], b[2], b[3]);
                }
            }
        }
        __syncwarp();
        if (it + S < steps) fetch(stage, page, slot);
        if (++stage == S) stage = 0, phase ^= 1;
    }
    if (!ok)  // a copy that has not landed in 2 s: leave none under way, and no number
        for (int i = 0; i < S; ++i) mbar_wait(&bar[i], phase ^ (i < stage));

    // ---- results
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[rt][e];
            sum += __shfl_xor_sync(kFull, sum, 1);
            sum += __shfl_xor_sync(kFull, sum, 2);
            if (!ok) sum = NAN;
            const int r = rt * 16 + (lane >> 2) + 8 * e;
            if (r >= nrows) continue;
            const int f = row0 + r, t = s.first + f / p.group, qh = h * p.group + f % p.group;
            const int64_t row = (int64_t)t * p.q_heads + qh;
            if (p.direct) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                T* out = static_cast<T*>(p.out) + t * p.o_tok + qh * p.o_head + 2 * (lane & 3);
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<uint32_t*>(out + n * 8) = pack2<T>(o[rt][n][2 * e] * inv, o[rt][n][2 * e + 1] * inv);
                if (p.lse && (lane & 3) == 0)
                    p.lse[row] = sum == 0.f ? -INFINITY : (m[rt][e] + log2f(sum)) * 0.69314718055994531f;
            } else {
                const int64_t at = (int64_t)part * p.tokens * p.q_heads + row;
                float* out = p.part_o + at * D + 2 * (lane & 3);
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[rt][n][2 * e], o[rt][n][2 * e + 1]);
                if ((lane & 3) == 0) p.part_ml[at] = make_float2(m[rt][e], sum);
            }
        }
}

// ------------------------------------------------------------------ joining the parts
// WPR warps a row, each with every WPR-th part: one where rows are many, 4 or 16 where parts are
// (147 parts of 64 rows: 63 us by one warp a row, latency after latency).  Bound: L2 (the parts were
// just written), so loads are 16 bytes a lane and eight parts are in flight.
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(WPR == 16 ? 512 : 128) attn_join_kernel(const AttnParams p) {
    constexpr int VE = D % 128 == 0 ? 4 : D % 64 == 0 ? 2 : 1, NV = D / (32 * VE);
    __shared__ float s_acc[WPR][D], s_sum[WPR], s_top[WPR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = WPR == 1 ? 0 : warp;
    const int64_t all = (int64_t)p.tokens * p.q_heads, row = WPR == 1 ? (int64_t)blockIdx.x * 4 + warp : blockIdx.x;
    pdl_wait();
    if (row >= all) return;
    const int t = (int)(row / p.q_heads), qh = (int)(row % p.q_heads);
    int np = p.prefix_splits, n;  // parts over the prefix, and all
    if (p.prefix_ctas > 0) {
        const int u = qh / p.group * p.prefix_tiles + (t * p.group + qh % p.group) / 256;
        np = prefix_cta(p, (u + 1) * p.prefix_steps - 1) - prefix_cta(p, u * p.prefix_steps) + 1;
    }
    n = np;
    if (p.own_chunks > 0) {
        const Sequence s = sequence(p, sequence_of_warp(p.q_indptr, p.rows, t));
        if (t >= s.first && t < s.first + s.asked) n += (s.len + p.own_chunk - 1) / p.own_chunk;
    }
    // lane l holds the maximum and sum of the l-th of 32 of the warp's parts at a time
    auto part = [&](int i) { return (i < np ? i : i - np + p.prefix_splits) * all + row; };
    const int count = (n - mine + WPR - 1) / WPR;
    float2 first = make_float2(-INFINITY, 0.f);
    if (lane < count) first = p.part_ml[part(lane * WPR + mine)];
    float top = first.x;
    for (int i = lane + 32; i < count; i += 32) top = fmaxf(top, p.part_ml[part(i * WPR + mine)].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, x));
    const float base = top == -INFINITY ? 0.f : top;
    float acc[NV * VE], sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV * VE; ++i) acc[i] = 0.f;
    for (int i0 = 0; i0 < count; i0 += 32) {
        float2 ml = first;
        if (i0 > 0) ml = i0 + lane < count ? p.part_ml[part((i0 + lane) * WPR + mine)] : make_float2(-INFINITY, 0.f);
        // 0: nothing seen there, nothing written; a NaN score leaves the sum NaN
        const float mine_f = ml.y == 0.f ? 0.f : ml.y != ml.y ? NAN : exp2_fast(ml.x - base);
        sum += mine_f == 0.f ? 0.f : mine_f * ml.y;
        const int here = min(32, count - i0);
#pragma unroll 8
        for (int i = 0; i < here; ++i) {
            const float f = __shfl_sync(kFull, mine_f, i);
            const float* x = p.part_o + part((i0 + i) * WPR + mine) * D;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float v[VE];
                if constexpr (VE == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(x + (j * 32 + lane) * 4);
                    v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
                } else if constexpr (VE == 2) {
                    const float2 y = *reinterpret_cast<const float2*>(x + (j * 32 + lane) * 2);
                    v[0] = y.x, v[1] = y.y;
                } else {
                    v[0] = x[j * 32 + lane];
                }
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[j * VE + e] += f == 0.f ? 0.f : f * v[e];
            }
        }
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(kFull, sum, x);
    if constexpr (WPR > 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VE; ++e) s_acc[warp][(j * 32 + lane) * VE + e] = acc[j * VE + e];
        if (lane == 0) s_sum[warp] = sum, s_top[warp] = top;
        __syncthreads();
        if (warp > 0) return;
        top = s_top[0];
#pragma unroll
        for (int w = 1; w < WPR; ++w) top = fmaxf(top, s_top[w]);
        const float all_base = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV * VE; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float f = s_sum[w] == 0.f ? 0.f : exp2_fast(s_top[w] - all_base);
            sum += f * s_sum[w];
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[j * VE + e] += f * s_acc[w][(j * 32 + lane) * VE + e];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(p.out) + t * p.o_tok + qh * p.o_head;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        T* y = out + (j * 32 + lane) * VE;
        if constexpr (VE == 4) {
            *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(acc[j * 4] * inv, acc[j * 4 + 1] * inv),
                                                      pack2<T>(acc[j * 4 + 2] * inv, acc[j * 4 + 3] * inv));
        } else if constexpr (VE == 2) {
            *reinterpret_cast<uint32_t*>(y) = pack2<T>(acc[j * 2] * inv, acc[j * 2 + 1] * inv);
        } else {
            *y = from_f32<T>(acc[j] * inv);
        }
    }
    if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

// At most eight parts, many rows: a warp joins four heads of a token.  What the chain of the sequence's place
// and length, m and l, and the sums costs is paid once for the four, and their loads are under way
// together (a warp a row: 92 us for 119,040 rows of three parts, 183 MB).
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_few_kernel(const AttnParams p) {
    constexpr int VE = D % 128 == 0 ? 4 : D % 64 == 0 ? 2 : 1, NV = D / (32 * VE), kHeads = 4, kParts = 8;
    const int lane = threadIdx.x & 31;
    const int groups = (p.q_heads + kHeads - 1) / kHeads;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), all = (int64_t)p.tokens * p.q_heads;
    const int t = (int)(id / groups), h0 = (int)(id % groups) * kHeads;
    pdl_wait();
    if (t >= p.tokens) return;
    int own = 0;
    if (p.own_chunks > 0) {
        const Sequence s = sequence(p, sequence_of_warp(p.q_indptr, p.rows, t));
        if (t >= s.first && t < s.first + s.asked) own = (s.len + p.own_chunk - 1) / p.own_chunk;
    }
    // lane 8 k + i: part i of head h0 + k
    const int h = min(h0 + lane / kParts, p.q_heads - 1), i = lane % kParts;
    int np = p.prefix_splits;  // parts over the prefix
    if (p.prefix_ctas > 0) {
        const int u = h / p.group * p.prefix_tiles + (t * p.group + h % p.group) / 256;
        np = prefix_cta(p, (u + 1) * p.prefix_steps - 1) - prefix_cta(p, u * p.prefix_steps) + 1;
    }
    const int n = np + own, place = i < np ? i : i - np + p.prefix_splits;
    const int64_t at = place * all + (int64_t)t * p.q_heads + h;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (i < n) ml = p.part_ml[at];
    float top = ml.x;
#pragma unroll
    for (int x = kParts / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, x));
    // 0: nothing seen there, nothing written; a NaN score leaves the sum NaN
    float f = ml.y == 0.f ? 0.f : ml.y != ml.y ? NAN : exp2_fast(ml.x - (top == -INFINITY ? 0.f : top));
    float sum = f == 0.f ? 0.f : f * ml.y;
#pragma unroll
    for (int x = kParts / 2; x; x >>= 1) sum += __shfl_xor_sync(kFull, sum, x);
    if (p.lse && i == 0 && h0 + lane / kParts < p.q_heads)
        p.lse[(int64_t)t * p.q_heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
    f *= sum == 0.f ? 0.f : 1.f / sum;
    float acc[kHeads][NV * VE];
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
#pragma unroll
        for (int e = 0; e < NV * VE; ++e) acc[k][e] = 0.f;
    const int most = __reduce_max_sync(kFull, n);
#pragma unroll 2
    for (int j = 0; j < most; ++j) {
        float v[kHeads][NV * VE], w[kHeads];
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            w[k] = __shfl_sync(kFull, f, k * kParts + j);
            const int64_t from = __shfl_sync(kFull, at, k * kParts + j);
            const float* x = p.part_o + from * D;
#pragma unroll
            for (int e = 0; e < NV * VE; ++e) v[k][e] = 0.f;
            if (w[k] != 0.f) {
#pragma unroll
                for (int q = 0; q < NV; ++q) {
                    if constexpr (VE == 4) {
                        const float4 y = *reinterpret_cast<const float4*>(x + (q * 32 + lane) * 4);
                        v[k][q * 4] = y.x, v[k][q * 4 + 1] = y.y, v[k][q * 4 + 2] = y.z, v[k][q * 4 + 3] = y.w;
                    } else if constexpr (VE == 2) {
                        const float2 y = *reinterpret_cast<const float2*>(x + (q * 32 + lane) * 2);
                        v[k][q * 2] = y.x, v[k][q * 2 + 1] = y.y;
                    } else {
                        v[k][q] = x[q * 32 + lane];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kHeads; ++k)
#pragma unroll
            for (int e = 0; e < NV * VE; ++e) acc[k][e] += w[k] * v[k][e];
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
        if (h0 + k >= p.q_heads) break;
        T* out = static_cast<T*>(p.out) + t * p.o_tok + (h0 + k) * p.o_head;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            T* y = out + (q * 32 + lane) * VE;
            if constexpr (VE == 4) {
                *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(acc[k][q * 4], acc[k][q * 4 + 1]),
                                                          pack2<T>(acc[k][q * 4 + 2], acc[k][q * 4 + 3]));
            } else if constexpr (VE == 2) {
                *reinterpret_cast<uint32_t*>(y) = pack2<T>(acc[k][q * 2], acc[k][q * 2 + 1]);
            } else {
                *y = from_f32<T>(acc[k][q]);
            }
        }
    }
}

// ------------------------------------------------------------------ host
// Bytes of own parts.  A prompt of 8192 tokens, 16 heads of 256 on 4: 4.4 ms with 256 MiB, 5.3 with 16
// chunks in 2 GiB.  256 sequences of 8 tokens and 500 keys, one of 65536: 0.46 ms with 32 chunks in 1 GiB,
// 0.45 with 64 in 2 GiB, 0.82 with 8 in 256 MiB; 1024 of 16 tokens with one such: 2.9 ms with 4 chunks, 2.2
// with 16 in 4 GiB.
constexpr int64_t kFewParts = 256ll << 20, kMostParts = 1ll << 30;

// Keys of a chunk so that the parts of `rows` rows take `bytes` at most (or are one for each row).
int64_t fit_chunk(int64_t max_seq, int64_t rows, int64_t bytes, int dim) {
    const int64_t parts = std::max<int64_t>(1, bytes / (std::max<int64_t>(1, rows) * (dim * 4 + 8)));
    return ceil_div(max_seq, parts * 16) * 16;
}

struct Plan {
    AttnParams p;
    int rt_own, rt_prefix;  // 16-row tiles of a CTA of the kernel for few rows; 0: the tcgen05 kernel
    int64_t own_units, prefix_units;
    size_t ws_bytes;   // what the call takes
    size_t ws_enough;  // what a call of these sizes or of any smaller ones takes at most
};

// Bytes of so many rows of parts: the sums, then m and l.
size_t sum_bytes(int64_t rows, int dim) { return ((size_t)rows * dim * sizeof(float) + 255) / 256 * 256; }
size_t parts_bytes(int64_t rows, int dim) { return sum_bytes(rows, dim) + ((size_t)rows * sizeof(float2) + 255) / 256 * 256; }

// CTAs of the tcgen05 kernel over the prefix, by the time that the whole call would take: a CTA,
// one on an SM, has its steps at 1.75 us (1.2 where there is one row tile), 10 us to begin and end
// (18 where the own parts keep the memory busy) and 8 for each pair of head and row tile that it
// goes on to; the SMs that they leave, and their time after them, go to the own parts (own_bytes at
// 6 TB/s, 12 us at least); and each part of a row is written and read once more.  As many CTAs for
// each pair, or fewer than pairs and even shares.  It finds the best of a sweep of 64 sequences of
// 540 keys behind 8192 (56 CTAs: 56 us; 32: 69, 128: 75), of 256 of 180 keys behind 32768 (128: 172; 64: 243,
// 144: 180) and of 48 of 5 tokens and 320 keys behind 5003 (96: 49; 64: 58, 128: 59).
void share_prefix(AttnParams& p, int64_t rows, int dim, double own_bytes) {
    const int64_t units = (int64_t)p.prefix_tiles * p.kv_heads;
    p.prefix_steps = (int)ceil_div(p.prefix_len, 128);
    p.prefix_work = (int)(units * p.prefix_steps);
    const double step = rows > 128 ? 1.75 : 1.2, begin = own_bytes > 0 ? 18.0 : 10.0;
    const double own = own_bytes > 0 ? std::max(own_bytes / 6e6, 12.0) : 0.0;
    double best = 1e30;
    int64_t ctas = 1;
    for (int64_t n = 1; n <= std::min<int64_t>(kSMs, p.prefix_work); ++n) {
        if (n > units && (n % units || n / units > p.prefix_steps)) continue;
        const double more = n >= units ? 0.0 : (double)(ceil_div(units, n) - (units % n == 0));
        const double cta = begin + step * (double)ceil_div(p.prefix_work, n) + 8.0 * more;
        const double all = own + cta * (double)n / kSMs;
        const double parts = n >= units ? (double)(n / units) : 1.0 + (double)n / (double)units;
        const double t = std::max(cta, all) + parts * (double)rows * p.kv_heads * dim * 8 / 6e6;
        if (t < best * 0.999) best = t, ctas = n;
    }
    p.prefix_ctas = (int)ctas;
    p.prefix_per_unit = ctas % units == 0 ? (int)(ctas / units) : 0;
    // a pair's steps lie in at most so many shares of at least prefix_work / ctas steps
    const int least = p.prefix_work / p.prefix_ctas;
    p.prefix_splits = p.prefix_per_unit ? p.prefix_per_unit : (p.prefix_steps + least - 2) / least + 1;
}

int make_plan(const tg_prefix_attention_args* a, Plan* plan, const char* op) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_cache(a->cache, op);
    if (rc == TG_OK && !a->pages) rc = set_error(TG_EINVAL, "%s: null page table", op);
    if (rc != TG_OK) return rc;
    const tg_paged_kv& c = *a->cache;
    const tg_csr& t = *a->pages;
    if (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 256)
        return set_error(TG_EUNSUPPORTED, "%s: head dim must be 64, 96, 128 or 256 (got %d)", op, c.dim);
    if (a->q_heads < 1 || a->q_heads % c.heads)
        return set_error(TG_EINVAL, "%s: q_heads (%d) must be a multiple of the cache's heads (%d)", op, a->q_heads,
                         c.heads);
    if (a->tokens < 0 || a->tokens > INT32_MAX || t.rows < 0 || t.rows > INT32_MAX || t.nnz < 0)
        return set_error(TG_EINVAL, "%s: bad size (tokens=%lld sequences=%lld pages=%lld)", op, (long long)a->tokens,
                         (long long)t.rows, (long long)t.nnz);
    if (a->prefix_len < 0 || a->n_prefix_pages < 0 || a->prefix_len > INT32_MAX / 2 ||
        ceil_div(a->prefix_len, c.page_size) > a->n_prefix_pages)
        return set_error(TG_EINVAL, "%s: prefix_len (%lld) must be in [0, 2^30) and inside its %lld pages of %lld", op,
                         (long long)a->prefix_len, (long long)a->n_prefix_pages, (long long)c.page_size);
    if (a->max_seq_len < 0 || a->max_q_len < 0)
        return set_error(TG_EINVAL, "%s: negative max_seq_len or max_q_len", op);
    if (a->q_indptr && a->tokens > 0 && a->max_q_len == 0)
        return set_error(TG_EINVAL, "%s: a max_q_len of 0 answers none of the %lld tokens", op, (long long)a->tokens);
    if (!(a->scale > 0.0) || a->scale > 1e30) return set_error(TG_EINVAL, "%s: scale must be positive", op);
    if (a->flags & ~(TG_FLAG_CAUSAL | TG_FLAG_BOUNDS_CHECK))
        return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if (a->prefix_len > 0 && c.pages == 0) return set_error(TG_EINVAL, "%s: a prefix in a cache without pages", op);
    if (a->tokens * (a->q_heads / c.heads) > INT32_MAX / 2)
        return set_error(TG_EUNSUPPORTED, "%s: too many rows for one launch", op);
    const int64_t slots = c.pages == 0 ? 0 : t.nnz > INT32_MAX / c.page_size ? INT32_MAX / 2 : t.nnz * c.page_size;
    const int64_t max_seq = std::min({a->max_seq_len, slots, (int64_t)INT32_MAX / 2});
    const int64_t max_q = a->q_indptr ? std::min(a->max_q_len, a->tokens) : 1;

    AttnParams& p = plan->p;
    p = {};
    p.q = a->q.data, p.k = c.k, p.v = c.v, p.out = a->out.data, p.lse = a->lse;
    p.q_tok = stride_of(a->tokens, a->q.token_stride), p.q_head = stride_of(a->q_heads, a->q.head_stride);
    p.o_tok = stride_of(a->tokens, a->out.token_stride), p.o_head = stride_of(a->q_heads, a->out.head_stride);
    p.k_page = stride_of(c.pages, c.k_page_stride), p.v_page = stride_of(c.pages, c.v_page_stride);
    p.k_slot = stride_of(c.page_size, c.k_slot_stride), p.v_slot = stride_of(c.page_size, c.v_slot_stride);
    p.k_head = stride_of(c.heads, c.k_head_stride), p.v_head = stride_of(c.heads, c.v_head_stride);
    p.pages = (int)c.pages, p.page_size = (int)c.page_size;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (c.page_size == (1ll << i)) p.page_shift = i;
    p.q_heads = a->q_heads, p.kv_heads = c.heads, p.group = a->q_heads / c.heads;
    p.tokens = (int)a->tokens, p.rows = (int)t.rows;
    p.q_indptr = a->q_indptr, p.indptr = t.indptr, p.indices = t.indices, p.seq_len = a->seq_len;
    p.prefix_pages = a->prefix_pages, p.nnz = t.nnz;
    p.max_seq = (int)max_seq, p.max_q = (int)max_q, p.prefix_len = (int)a->prefix_len;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.causal = (a->flags & TG_FLAG_CAUSAL) != 0;

    // The kernel for few rows reads the keys once for each 32 rows, the tcgen05 kernel once for
    // each 256 (it exists for heads of 64 and 128) but begins and ends for 10 us.  Own parts of 320
    // keys, 48 sequences: 56 rows 58 against 64 us, 80 rows 79 against 74 us.  A prefix of 16384
    // keys: 40 rows 60 against 39 us, 64 rows 64 against 37 us (one of 2000: 29 against 35).
    const int64_t rows_own = max_q * p.group, rows_all = a->tokens * p.group;
    const bool tc = c.dim == 64 || c.dim == 128;
    plan->rt_own = tc && rows_own > 64 ? 0 : rows_own > 16 && c.dim <= 128 ? 2 : 1;
    plan->rt_prefix = tc && rows_all > 32 ? 0 : rows_all > 16 && c.dim <= 128 ? 2 : 1;
    if (p.prefix_len > 0 && plan->rt_prefix) plan->rt_own = plan->rt_prefix;  // one launch for both
    const int64_t warps = kSMs * 7;  // warps of the kernel for few rows that run at once (heads of 128)
    const int64_t tiles_own = ceil_div(std::max<int64_t>(rows_own, 1), plan->rt_own ? 16 * plan->rt_own : 256);
    const int64_t tiles_all = ceil_div(std::max<int64_t>(rows_all, 1), plan->rt_prefix ? 16 * plan->rt_prefix : 256);
    if (p.prefix_len > 0) {
        p.prefix_tiles = (int)tiles_all;
        if (plan->rt_prefix) {
            const int64_t n = std::max<int64_t>(1, warps / (tiles_all * c.heads));
            p.prefix_chunk = (int)std::max<int64_t>(128, ceil_div(ceil_div(p.prefix_len, n), 16) * 16);
            p.prefix_splits = (int)ceil_div(p.prefix_len, p.prefix_chunk);
        } else {
            if (tiles_all * c.heads > INT32_MAX / ceil_div(p.prefix_len, 128))
                return set_error(TG_EUNSUPPORTED, "%s: too many rows for one launch", op);
            share_prefix(p, rows_all, c.dim, (double)t.nnz * c.page_size * c.heads * c.dim * 4);
        }
    }
    if (max_seq > 0 || p.prefix_len == 0) {
        // The kernel for few rows: two rounds of its warps, in chunks of 256 to 512 keys (or 64
        // chunks, for sequences that may be long; 16 where sequences and heads alone make two rounds,
        // as each chunk costs workspace) so that long sequences do not end alone.  One
        // sequence of 32768 keys: 34 us in chunks of 256, 38 in chunks of 128 (the join has 256
        // parts); 64 sequences of 4096: 184 to 188 us for any bounds from 128 to 1024.  The tcgen05
        // kernel: two pieces an SM.
        const int64_t units = std::max<int64_t>(1, t.rows * tiles_own * c.heads), part_rows = a->tokens * a->q_heads;
        if (plan->rt_own) {
            const int64_t even = ceil_div(ceil_div(max_seq, std::max<int64_t>(1, 2 * warps / units)), 16) * 16;
            const int64_t most = units >= 2 * warps ? 16 : 64;
            p.own_chunk = (int)std::min(std::max<int64_t>(256, even), std::max<int64_t>(512, ceil_div(max_seq, most * 16) * 16));
            // Chunks of every sequence have their place in the workspace, as many as the longest may
            // have.  Above kFewParts chunks grow until it fits there, but not beyond what even shares
            // of all listed keys would be; above kMostParts they grow whatever it costs.
            const int64_t keys = std::min(slots, t.rows * max_seq);
            const double share = (double)keys * tiles_own * c.heads / (2 * warps);
            const int64_t few = fit_chunk(max_seq, part_rows, kFewParts, c.dim);
            const int64_t chunk = std::max({(int64_t)p.own_chunk, share < (double)few ? ((int64_t)share + 15) / 16 * 16 : few,
                                            fit_chunk(max_seq, part_rows, kMostParts, c.dim)});
            p.own_chunk = (int)chunk;
        } else {
            const int64_t n = std::max<int64_t>(1, 2 * kSMs / units);
            const int64_t most = fit_chunk(max_seq, part_rows, kMostParts, c.dim);  // many tokens of no sequence
            p.own_chunk = (int)std::max<int64_t>(256, ceil_div(std::max(ceil_div(max_seq, n), most), 128) * 128);
        }
        p.own_chunks = (int)std::max<int64_t>(1, ceil_div(max_seq, p.own_chunk));
    }
    plan->own_units = t.rows * tiles_own * p.own_chunks;
    plan->prefix_units = p.prefix_ctas ? p.prefix_ctas : tiles_all * p.prefix_splits;
    if ((plan->own_units + plan->prefix_units) * c.heads > INT32_MAX - kSMs || c.heads > 65535)
        return set_error(TG_EUNSUPPORTED, "%s: too many rows for one launch", op);
    p.tiles = (int)tiles_own;
    p.own_pieces = (int)(plan->own_units * c.heads);
    const int parts = p.prefix_splits + p.own_chunks;
    p.direct = parts == 1;
    p.fill = p.direct && p.q_indptr && p.prefix_len == 0;
    const int64_t rows = a->tokens * a->q_heads;
    plan->ws_bytes = p.direct ? 0 : parts_bytes(parts * rows, c.dim);
    // Fewer sequences or listed pages are cut into more parts, so what this call takes is no bound for
    // smaller ones.  A part has 128 keys of the prefix or 256 own keys, or the last of them.  Over the
    // prefix, more than two parts of a row are one for each of so many warps (or CTAs) that together
    // have 32 (or 256) rows each; own parts fit kMostParts.
    const int64_t of_prefix = ceil_div(p.prefix_len, 128), of_own = ceil_div(max_seq, 256);
    const int64_t prefix_rows = std::min(of_prefix * rows, std::max<int64_t>({2 * rows, warps * 32, (int64_t)kSMs * 256}));
    const int64_t own_rows = std::min(of_own * rows, std::max<int64_t>(rows, kMostParts / (c.dim * 4 + 8)));
    plan->ws_enough = of_prefix + of_own <= 1 ? 0 : parts_bytes(prefix_rows + own_rows, c.dim);
    return TG_OK;
}

template <typename T, int D, int RT>
int rows_launch(const AttnParams& p, int64_t units, bool pdl, cudaStream_t st) {
    using C = RowCfg<D, RT>;
    auto kernel = p.fill ? attn_rows_kernel<T, D, RT, true> : attn_rows_kernel<T, D, RT, false>;
    const int box = std::gcd(p.page_size, kStepKeys);
    CUtensorMap kmap, vmap;
    int rc = cache_maps(p, std::is_same<T, __half>::value, D, box, &kmap, &vmap);
    if (rc != TG_OK) return rc;
    rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                              "cudaFuncSetAttribute");
    if (rc != TG_OK) return rc;
    const dim3 grid((unsigned)units, (unsigned)p.kv_heads);
    if (pdl) return launch_pdl("attn_rows_kernel", kernel, grid, 32, C::kSmem, st, p, box, kmap, vmap);
    kernel<<<grid, 32, C::kSmem, st>>>(p, box, kmap, vmap);
    return check_launch("attn_rows_kernel");
}

template <typename T, int D>
int attn_run(const Plan& plan, void* ws, cudaStream_t st) {
    AttnParams p = plan.p;
    const size_t rows = (size_t)p.tokens * p.q_heads;
    const size_t parts = p.prefix_splits + p.own_chunks;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + sum_bytes((int64_t)(parts * rows), D));
    int rc = TG_OK;
    bool second = false;
    if (p.prefix_ctas > 0) {
        if constexpr (D == 64 || D == 128) {
            AttnParams q = p;
            q.over_prefix = 1;
            q.tiles = p.prefix_tiles;
            rc = attn_tc_run<T>(q, D, p.prefix_ctas, false, st);
        }
        second = true;
    } else {
        p.prefix_units = (int)plan.prefix_units;
    }
    const int64_t units = plan.own_units + p.prefix_units;
    if (rc == TG_OK && units > 0) {
        if (plan.rt_own == 0) {
            if constexpr (D == 64 || D == 128) rc = attn_tc_run<T>(p, D, std::min(p.own_pieces, kSMs), second, st);
        } else if (plan.rt_own == 2) {
            if constexpr (D <= 128) rc = rows_launch<T, D, 2>(p, units, second, st);
        } else {
            rc = rows_launch<T, D, 1>(p, units, second, st);
        }
    }
    if (rc != TG_OK) return rc;
    if (p.direct) return TG_OK;
    // Four heads a warp, for many rows: 119,040 of 3 parts 38 us against 92 with a warp a row; 8192 of
    // 5 parts do better with a warp each (167 against 174 us for the call).
    if (parts <= 8 && rows >= (size_t)kSMs * 128) {
        const int64_t warps = p.tokens * ceil_div(p.q_heads, 4);
        return launch_pdl("attn_join_few_kernel", attn_join_few_kernel<T, D>, dim3((unsigned)ceil_div(warps, 4)), 128, 0, st, p);
    }
    // 64 rows of 130 parts: 99 us for the call with 16 warps a row, 102 with 4.
    if (parts > 32 && rows < kSMs * 8)
        return launch_pdl("attn_join_kernel", attn_join_kernel<T, D, 16>, dim3((unsigned)rows), 512, 0, st, p);
    if (parts > 8 && rows < 4 * kSMs * 16)
        return launch_pdl("attn_join_kernel", attn_join_kernel<T, D, 4>, dim3((unsigned)rows), 128, 0, st, p);
    return launch_pdl("attn_join_kernel", attn_join_kernel<T, D, 1>, dim3((unsigned)ceil_div((int64_t)rows, 4)), 128, 0, st, p);
}

template <typename T>
int attention(const tg_prefix_attention_args* a, void* ws, size_t ws_bytes, tg_stream_t stream, const char* op) {
    Plan plan;
    int rc = make_plan(a, &plan, op);
    if (rc == TG_OK) rc = check_table(a->pages, a->cache, a->tokens, a->q_indptr, a->seq_len, op);
    if (rc != TG_OK) return rc;
    if (a->tokens == 0) return TG_OK;
    const tg_paged_kv& c = *a->cache;
    if (!a->q.data || !a->out.data) return set_error(TG_EINVAL, "%s: null q/out", op);
    if (a->prefix_len > 0 && !a->prefix_pages) return set_error(TG_EINVAL, "%s: null prefix_pages", op);
    const uint64_t at = reinterpret_cast<uint64_t>(a->q.data) | reinterpret_cast<uint64_t>(a->out.data) |
                        reinterpret_cast<uint64_t>(c.k) | reinterpret_cast<uint64_t>(c.v);
    const AttnParams& p = plan.p;
    const uint64_t strides = (uint64_t)(p.q_tok | p.q_head | p.o_tok | p.o_head | p.k_page | p.k_slot | p.k_head |
                                        p.v_page | p.v_slot | p.v_head);
    if (at % 16 || strides % 8)
        return set_error(TG_EINVAL, "%s: rows must be 16-byte aligned (strides multiples of 8 elements)", op);
    if (ws_bytes < plan.ws_bytes || (plan.ws_bytes && !ws))
        return set_error(TG_ENOMEM, "%s: workspace of %zu bytes, %zu needed", op, ws ? ws_bytes : (size_t)0,
                         plan.ws_bytes);
    if (reinterpret_cast<uint64_t>(ws) % 16)
        return set_error(TG_EINVAL, "%s: the workspace must be 16-byte aligned", op);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->flags & TG_FLAG_BOUNDS_CHECK) {
        rc = paged_bounds_check(*a->pages, c.page_size, a->seq_len, a->max_seq_len, a->tokens, a->q_indptr,
                                a->q_indptr ? a->max_q_len : 1, a->prefix_pages, ceil_div(a->prefix_len, c.page_size),
                                false, op, st);
        if (rc != TG_OK) return rc;
    }
    switch (c.dim) {
        case 64: return attn_run<T, 64>(plan, ws, st);
        case 96: return attn_run<T, 96>(plan, ws, st);
        case 128: return attn_run<T, 128>(plan, ws, st);
        default: return attn_run<T, 256>(plan, ws, st);
    }
}

}  // namespace
}  // namespace tg

extern "C" {

size_t tg_prefix_attention_workspace_bytes(const tg_prefix_attention_args* a) {
    tg::Plan plan;
    return tg::make_plan(a, &plan, "tg_prefix_attention") == TG_OK ? plan.ws_enough : 0;
}

size_t tg_prefix_attention_needed_bytes(const tg_prefix_attention_args* a) {
    tg::Plan plan;
    return tg::make_plan(a, &plan, "tg_prefix_attention") == TG_OK ? plan.ws_bytes : 0;
}

int tg_prefix_attention_f16(const tg_prefix_attention_args* a, void* workspace, size_t workspace_bytes,
                            tg_stream_t stream) {
    return tg::attention<__half>(a, workspace, workspace_bytes, stream, "tg_prefix_attention_f16");
}

int tg_prefix_attention_bf16(const tg_prefix_attention_args* a, void* workspace, size_t workspace_bytes,
                             tg_stream_t stream) {
    return tg::attention<__nv_bfloat16>(a, workspace, workspace_bytes, stream, "tg_prefix_attention_bf16");
}

}  // extern "C"
