// Attention of many rows at once (tcgen05): the shared prefix of a batch of more than a few
// rows, and sequences with many query tokens.
//
// A CTA takes up to 256 rows (two tiles of 128) of one key head and a range of keys, 128 at a
// time.  S = Q K^T of a tile lands in TMEM; the tile's warpgroup (one thread a row, so neither
// the maximum nor the sum crosses lanes) turns it into P, writes P over S in the values' type,
// and O += P V reads P from there.  While one tile's softmax runs, the tensor core works for
// the other.
//
//   TMEM columns      [0,128) S0/P0   [128,256) S1/P1   [256,256+D) O0   [384,384+D) O1
//   warps 0-3, 4-7    softmax of tile 0, 1: S -> P, the running maximum and sum, O at the end
//   warps 8, 10       fetch K, V tiles into a ring of shared memory by TMA, in boxes of as many
//                     rows as divide both a page and a tile
//   warp 9            issues the matrix instructions
//   warp 11           how many keys each row sees
//
// Bound: Q K^T reads both operands from shared memory, 8 KB for 64 cycles of arithmetic, and gets
// 107 bytes a cycle; with P V (P from TMEM) and the tiles' arrival that is 2500 cycles for 128 keys
// of two tiles, of 3200 that a step takes; the rest is the chain S, maximum, P, product of a tile
// where the other tile does not cover it.  4608 rows of each of 8 key heads of 128 over 16384 keys:
// 270 us, 1.14 PFLOP/s, 69 % of the library product's burst; tensor pipe 63 % active, special-function
// unit 64 %, issue slots 38 %.
//
// O is rescaled only where a row's maximum has grown by more than 2^8 since the value that P is
// taken relative to: P stays below 2^8 (2^15 in float16, where the largest weight is at least 2^7, so
// that small weights keep their bits: what they may lose is keys * 2^-32 of the largest value),
// inside the range of either type and of the 32-bit sums, and the relative precision of P is that of
// any other reference.
#include <numeric>

#include "tg_tcgen05.cuh"

namespace tg {
namespace {

constexpr int kTile = 128;   // rows of a tile, keys of a step
constexpr int kThreads = 384;
constexpr uint32_t kCols = 512;
constexpr uint32_t kColO = 256;
constexpr float kGrow = 8.f;  // log2 of how far the maximum may grow before P is taken relative to a new one
constexpr int kLift = 7;      // float16: log2 of the largest P at first
constexpr int kFirst = 64;  // columns of P that are multiplied while the others are made

template <int D>
struct TcCfg {
    static constexpr int kBlock = kTile * D * 2;  // bytes of a tile of Q, K or V
    static constexpr int kHalf = kTile * 128;     // of 64 of its columns
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr int kSmem = (2 + kStages) * kBlock + 2048;  // and a TcShared
};

struct TcShared {
    uint64_t q_full[2], full[8], empty[8], s_full[2], p_half[2], p_full[2], o_done[2], seen_full, seen_free, tail, drained;
    uint32_t tmem;
    int fail;  // a wait ran out
    int seen[2 * kTile];
};

// Up to 256 rows over a range of keys, as all warps of a CTA see it.
struct Segment {
    Sequence s;
    const int64_t* list;
    int h, part, row0, nrows, k0, k1, keys, steps, ntiles;
};

// Row r of the segment, which sees the keys up to n, the long way, by a warp: only for a row that
// does not see a value that is not finite while others of its tile do.  (Inlined: a call would put
// the parameters on the stack of every thread.)
template <typename T, int D>
__device__ __forceinline__ void row_alone(const AttnParams& p, const Segment& g, int r, int n) {
    constexpr int E = D / 32;  // elements of a lane
    const int lane = threadIdx.x & 31, f = g.row0 + r, t = g.s.first + f / p.group, qh = g.h * p.group + f % p.group;
    const T* q = static_cast<const T*>(p.q) + t * p.q_tok + qh * p.q_head;
    float x[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32(q[lane * E + e]), acc[e] = 0.f;
    for (int key = g.k0; key < n; ++key) {
        int page, slot;
        locate(p, g.list, key, page, slot);
        const T* kr = static_cast<const T*>(p.k) + g.h * p.k_head + page * p.k_page + slot * p.k_slot + lane * E;
        const T* vr = static_cast<const T*>(p.v) + g.h * p.v_head + page * p.v_page + slot * p.v_slot + lane * E;
        float s = 0.f;
        if (page >= 0)
#pragma unroll
            for (int e = 0; e < E; ++e) s += x[e] * to_f32(kr[e]);
#pragma unroll
        for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(kFull, s, i);
        s *= p.scale_log2;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float keep = exp2_fast(m - base), w = exp2_fast(s - base);
        m = mn;
        l = l * keep + w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + (page >= 0 ? w * to_f32(vr[e]) : 0.f);
    }
    const int64_t at = (int64_t)t * p.q_heads + qh, pat = (int64_t)g.part * p.tokens * p.q_heads + at;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (p.direct) static_cast<T*>(p.out)[t * p.o_tok + qh * p.o_head + lane * E + e] = from_f32<T>(acc[e] * inv);
        else p.part_o[pat * D + lane * E + e] = acc[e];
    }
    if (lane == 0) {
        if (!p.direct) p.part_ml[pat] = make_float2(m, l);
        else if (p.lse) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
}

// The CTA's segments, one after the other, so that the keys of the next are under way while the
// results of one are written.  Over the prefix a CTA has a share of the steps of the (head, row
// tile) pairs; it may end one pair and begin another, and the parts of a pair are numbered by CTA.
// Over own pages it has every gridDim.x-th of the pieces (head, chunk, row tile, sequence), the
// last rows first: they see the most keys, and rounds of the CTAs are of like length.
struct Segments {
    int at, end;
    __device__ __forceinline__ explicit Segments(const AttnParams& p) {
        at = p.over_prefix ? prefix_start(p, blockIdx.x) : blockIdx.x;
        end = p.over_prefix ? prefix_start(p, blockIdx.x + 1) : p.own_pieces;
    }
    __device__ __forceinline__ bool next(const AttnParams& p, Segment& g) {
        for (;;) {
            if (at >= end) return false;
            if (p.over_prefix) {
                const int u = at / p.prefix_steps, first = at - u * p.prefix_steps;
                g.steps = min(p.prefix_steps - first, end - at);
                at += g.steps;
                g.h = u / p.tiles;
                g.row0 = (u - g.h * p.tiles) * 2 * kTile;
                g.part = blockIdx.x - prefix_cta(p, u * p.prefix_steps);
                g.s.first = 0;
                g.s.n = g.s.asked = p.tokens;
                g.nrows = min(p.tokens * p.group - g.row0, 2 * kTile);
                g.list = p.prefix_pages;
                g.keys = p.prefix_len;
                g.k0 = first * kTile;
                g.k1 = min(g.keys, g.k0 + g.steps * kTile);
            } else {
                int x = at;
                at += gridDim.x;
                g.h = x % p.kv_heads, x /= p.kv_heads;
                const int c = x % p.own_chunks;
                x /= p.own_chunks;
                const int b = x % p.rows;
                g.row0 = (p.tiles - 1 - x / p.rows) * 2 * kTile;
                g.s = sequence(p, b);
                g.nrows = min(g.s.asked * p.group - g.row0, 2 * kTile);
                g.list = p.indices + g.s.page0;
                g.keys = g.s.len;
                g.k0 = c * p.own_chunk;
                g.part = p.prefix_splits + c;
                // no rows, or no such chunk (the join does not ask for it)
                if (g.nrows <= 0 || (g.k0 >= g.keys && !p.direct)) continue;
                // no row sees more than the last one
                g.k1 = min(min(g.keys, g.k0 + p.own_chunk), keys_seen(p, g.s, (g.row0 + g.nrows - 1) / p.group, g.keys, g.keys));
                g.steps = g.k1 > g.k0 ? (g.k1 - g.k0 + kTile - 1) / kTile : 0;
            }
            g.ntiles = g.nrows > kTile ? 2 : 1;
            return true;
        }
    }
};

template <typename T, int D, bool FILL>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const AttnParams p, const int box,
                                                              const __grid_constant__ CUtensorMap kmap,
                                                              const __grid_constant__ CUtensorMap vmap) {
    using C = TcCfg<D>;
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(1024) unsigned char smem[];
    TcShared& sh = *reinterpret_cast<TcShared*>(smem + (2 + C::kStages) * C::kBlock);
    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    pdl_trigger();
    struct AtEnd {
        const AttnParams& p;
        __device__ ~AtEnd() {
            if constexpr (FILL)
                fill_unanswered<T, D>(p, blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), gridDim.x * (kThreads / 32));
            // grids of a call complete in order: this one, if it is the second, ends after the first
            if (blockIdx.x == 0) pdl_wait();
        }
    } at_end{p};
    if (!p.over_prefix) {
        Segments some(p);
        Segment g;
        if (!some.next(p, g)) return;
    }

    const uint32_t sq = smem_addr(smem), ring = sq + 2 * C::kBlock;
    const uint32_t b_q = smem_addr(sh.q_full), b_full = smem_addr(sh.full), b_empty = smem_addr(sh.empty),
                   b_s = smem_addr(sh.s_full), b_ph = smem_addr(sh.p_half), b_p = smem_addr(sh.p_full),
                   b_o = smem_addr(sh.o_done);
    volatile int* fail = &sh.fail;

    if (warp == 9) {
        tmem_alloc(smem_addr(&sh.tmem), kCols);
        if (lane == 0) {
            for (int i = 0; i < C::kStages; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.q_full[i], kTile);
                mbar_init(&sh.s_full[i], 1);
                mbar_init(&sh.p_half[i], kTile);
                mbar_init(&sh.p_full[i], kTile);
                mbar_init(&sh.o_done[i], 1);
            }
            mbar_init(&sh.seen_full, 32);
            mbar_init(&sh.seen_free, 2 * kTile);
            mbar_init(&sh.tail, 1);
            mbar_init(&sh.drained, 1);
            sh.fail = 0;
            fence_mbar_init();
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    Segments segments(p);
    Segment g;

    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0 : 1;
        constexpr uint32_t kBase = 1u << 4 | kType << 7 | kType << 10 | (kTile / 16) << 24;
        constexpr uint32_t kQK = kBase | (kTile / 8) << 17;
        constexpr uint32_t kPV = kBase | 1u << 16 | (D / 8) << 17;
        auto qk = [&](int i, int fill) {
            const uint32_t q = sq + i * C::kBlock, k = ring + fill % C::kStages * C::kBlock;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = (kk >> 2) * C::kHalf + (kk & 3) * 32;
                mma_ss(tmem + i * kTile, operand(q + off, 16), operand(k + off, 16), kQK, kk > 0);
            }
            commit(b_s + i * 8);
        };
        auto full = [&](int fill) {
            const bool ok = wait_warp(b_full + fill % C::kStages * 8, fill / C::kStages & 1, fail);
            fence_after();
            return ok;
        };
        auto holds = [&](uint32_t bar, int parity) { return wait_warp(bar, parity & 1, fail); };
        bool ok = true;
        int f = 0, done0 = 0, done1 = 0, seg0 = 0, seg1 = 0;  // fills; steps and segments of each tile
        while (ok && segments.next(p, g)) {
            if (g.steps == 0) continue;
            ok = holds(b_q, seg0++) && (g.ntiles == 1 || holds(b_q + 8, seg1++)) && full(f);
            if (!ok) break;
            for (int i = 0; i < g.ntiles; ++i) qk(i, f);
            commit(b_empty + f % C::kStages * 8);
            for (int j = 0; j < g.steps; ++j) {
                const int fv = f + 2 * j + 1, fk = fv + 1;
                const bool more = j + 1 < g.steps;
                ok = full(fv);
                const uint32_t v = ring + fv % C::kStages * C::kBlock;
                for (int i = 0; ok && i < g.ntiles; ++i) {
                    const int turn = (i ? done1 : done0) + j;
                    // the first columns of P are multiplied while the others are made
#pragma unroll
                    for (int kk = 0; kk < kTile / 16; ++kk) {
                        if (kk == 0 || kk == kFirst / 16) {
                            if (!(ok = holds((kk ? b_p : b_ph) + i * 8, turn))) break;
                            fence_after();
                        }
                        mma_ts(tmem + kColO + i * kTile, tmem + i * kTile + kk * 8, operand(v + kk * 2048, C::kHalf), kPV,
                               j > 0 || kk > 0);
                    }
                    if (!ok) break;
                    commit(b_o + i * 8);
                    // S of the next step goes over P: the tensor core works in the order of issue
                    if (more && i == 0 && !(ok = full(fk))) break;
                    if (more) qk(i, fk);
                }
                if (!ok) break;
                commit(b_empty + fv % C::kStages * 8);
                if (more) commit(b_empty + fk % C::kStages * 8);
            }
            f += 2 * g.steps;
            done0 += g.steps;
            if (g.ntiles == 2) done1 += g.steps;
        }
        if (!ok) {  // leave no product under way
            commit(smem_addr(&sh.drained));
            mbar_wait(&sh.drained, 0);
        }
    } else if (warp == 8 || warp == 10) {
        // Lane l looks up the page of box l of a tile one tile ahead; the warp issues box after
        // box.  A box past the end is not fetched; a page that does not exist is fetched from behind
        // the last one, which reads as zeros.
        const int is_v = warp == 10, boxes = kTile / box;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        int f0 = 0, tails = 0;  // fills before this segment, tails so far
        bool ok = true;
        while (ok && segments.next(p, g)) {
            int page, slot;
            auto find = [&](int at) {
                page = -1, slot = 0;
                if (at < g.k1) {
                    locate(p, g.list, at, page, slot);
                    if (page < 0) page = p.pages;
                }
            };
            if (lane < boxes) find(g.k0 + lane * box);
            for (int j = 0; j < g.steps; ++j) {
                const int f = f0 + 2 * j + is_v, st = f % C::kStages, kt = g.k0 + j * kTile, have = min(g.k1 - kt, kTile);
                const uint32_t dst = ring + st * C::kBlock, bar = b_full + st * 8;
                // Values past the end must be zeros (P is zero there, but 0 * NaN is not), so the
                // last tile lands on a barrier of its own and is delivered when they are.
                const bool tail = is_v && have < kTile;
                if (f >= C::kStages && !(ok = wait_warp(b_empty + st * 8, (f / C::kStages - 1) & 1, fail))) break;
                uint64_t* const land = tail ? &sh.tail : &sh.full[st];
                for (int b = 0; b < boxes; b += 32) {  // more than 32: page and tile have fewer than 4 rows in common
                    if (b > 0) find(kt + (b + lane) * box);
                    const uint32_t held = __ballot_sync(kFull, lane < boxes - b && page >= 0);
                    // the phase's one arrival comes with the last boxes: none completes it before
                    if (lane == 0) {
                        const uint32_t bytes = __popc(held) * box * D * 2;
                        if (b + 32 >= boxes) mbar_arrive_expect_tx(land, bytes);
                        else mbar_expect_tx(land, bytes);
                    }
                    __syncwarp();
                    for (int i = 0; i < min(boxes - b, 32); ++i) {
                        const int pg = __shfl_sync(kFull, page, i), sl = __shfl_sync(kFull, slot, i);
                        if (!(held >> i & 1)) continue;
#pragma unroll
                        for (int half = 0; half < D / 64; ++half)
                            load_box(dst + half * C::kHalf + (b + i) * box * 128, map, half * 64, sl, g.h, pg, smem_addr(land));
                    }
                }
                if (lane < boxes) find(kt + kTile + lane * box);
                if (tail) {
                    wait_warp(smem_addr(&sh.tail), tails++ & 1, fail);
                    for (int i = have * 8 + lane; i < kTile * 8; i += 32)
#pragma unroll
                        for (int half = 0; half < D / 64; ++half)
                            *reinterpret_cast<uint4*>(smem + (dst - sq) + half * C::kHalf + i * 16) = make_uint4(0, 0, 0, 0);
                    fence_async();
                    __syncwarp();
                    if (lane == 0) arrive(bar);
                }
            }
            if (ok) f0 += 2 * g.steps;
        }
        __syncwarp();
        if (*fail)  // leave no copy under way
            for (int f = max(0, f0 - C::kStages); f < f0 + C::kStages; ++f)
                if ((f & 1) == is_v) mbar_wait_brief(&sh.full[f % C::kStages], f / C::kStages & 1);
    } else if (warp == 11) {
        // Keys that each row sees, up to the segment's end: eight rows a lane, the searches of four
        // side by side.
        int turn = 0;
        bool ok = true;
        while (ok && segments.next(p, g)) {
            if (g.steps == 0) continue;
            if (turn > 0) ok = wait_warp(smem_addr(&sh.seen_free), (turn - 1) & 1, fail);
#pragma unroll 1
            for (int r0 = lane; r0 < 2 * kTile; r0 += 4 * 32) {
                int seen[4];
                if (p.over_prefix && (p.causal || p.q_indptr)) {
                    int t[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = r0 + i * 32;
                        t[i] = (g.row0 + (r < g.nrows ? r : 0)) / p.group;
                        lo[i] = p.q_indptr ? 0 : t[i];
                    }
                    if (p.q_indptr) {  // the last lo with q_indptr[lo] <= t
                        for (int step = 1 << (31 - __clz(p.rows)); step > 0; step >>= 1)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (lo[i] + step < p.rows && p.q_indptr[lo[i] + step] <= t[i]) lo[i] += step;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) seen[i] = prefix_seen(p, sequence(p, lo[i]), t[i], g.keys);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        seen[i] = p.over_prefix ? g.keys : keys_seen(p, g.s, (g.row0 + r0 + i * 32) / p.group, g.keys, g.keys);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = r0 + i * 32;
                    sh.seen[r] = r < g.nrows ? max(min(seen[i], g.k1), 0) : 0;
                }
            }
            arrive(smem_addr(&sh.seen_full));
            ++turn;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int my = warp >> 2, quarter = warp & 3, row = tid;  // tile, 32 rows of it, row of the CTA
        const uint32_t lanes = (uint32_t)quarter << 21;           // the warp's TMEM lanes, in bits 16-31
        const uint32_t ts = tmem + my * kTile + lanes, to = tmem + kColO + my * kTile + lanes;
        int done = 0, turn = 0;  // steps of the tile so far, segments
        while (segments.next(p, g)) {
            if (my >= g.ntiles) {
                if (g.steps > 0) {
                    wait_warp(smem_addr(&sh.seen_full), turn++ & 1, fail);
                    arrive(smem_addr(&sh.seen_free));
                }
                continue;
            }
            const int h = g.h, row0 = g.row0, nrows = g.nrows, steps = g.steps, k0 = g.k0, k1 = g.k1, first = g.s.first;
            int seen = 0;
            bool ok = true;
            if (steps > 0) {
                // ---- queries, swizzled, zeros where there is no row; all loads are under way at once
                constexpr int kStep = kTile / CH;  // rows between a thread's chunks
                const int rt = tid & (kTile - 1), c = rt % CH, f0 = my * kTile + rt / CH;
                const int dt = kStep / p.group, dg = kStep % p.group;
                int t = (row0 + f0) / p.group, x = (row0 + f0) % p.group;
                const char* q = static_cast<const char*>(p.q) + (first * p.q_tok + (int64_t)h * p.group * p.q_head) * 2 + c * 16;
                uint4 v[CH];
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const bool there = f0 + i * kStep < nrows;
                    v[i] = __ldg(reinterpret_cast<const uint4*>(q + (there ? (t * p.q_tok + x * p.q_head) * 2 : 0)));
                    t += dt;
                    x += dg;
                    if (x >= p.group) x -= p.group, ++t;
                }
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int r = rt / CH + i * kStep;
                    if (f0 + i * kStep >= nrows) v[i] = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(smem + my * C::kBlock + (c >> 3) * C::kHalf + r * 128 + (((c ^ r) & 7) << 4)) = v[i];
                }
                fence_async();
                arrive(b_q + my * 8);
                ok = wait_warp(smem_addr(&sh.seen_full), turn++ & 1, fail);
                seen = sh.seen[row];
                arrive(smem_addr(&sh.seen_free));
            }
            const bool rows_here = quarter * 32 + my * kTile < nrows;  // the warp has a row
            float m = -INFINITY, l = 0.f;                              // P is taken relative to m
            for (int j = 0; ok && j < steps; ++j) {
                if (!(ok = wait_warp(b_s + my * 8, (done + j) & 1, fail))) break;
                fence_after();
                if (rows_here) {
                    uint32_t x[kTile];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, x + c * 32);
                    wait_ld();
                    const int vis = seen - (k0 + j * kTile);
                    const bool cut = __any_sync(kFull, vis < kTile);
                    if (cut) {
#pragma unroll
                        for (int c = 0; c < kTile; ++c)
                            if (c >= vis) x[c] = 0xff800000u;  // -inf
                    }
                    float a0 = -INFINITY, a1 = -INFINITY, a2 = -INFINITY, a3 = -INFINITY;
#pragma unroll
                    for (int c = 0; c < kTile; c += 8) {
                        a0 = max3(a0, __uint_as_float(x[c]), __uint_as_float(x[c + 1]));
                        a1 = max3(a1, __uint_as_float(x[c + 2]), __uint_as_float(x[c + 3]));
                        a2 = max3(a2, __uint_as_float(x[c + 4]), __uint_as_float(x[c + 5]));
                        a3 = max3(a3, __uint_as_float(x[c + 6]), __uint_as_float(x[c + 7]));
                    }
                    const float top = max3(max3(a0, a1, a2), a3, a3) * p.scale_log2;
                    const float ref = reference<T, kLift>(top);
                    const bool grow = ref > m + kGrow || (m == -INFINITY && ref > m);
                    if (__any_sync(kFull, grow)) {
                        const float keep = grow ? exp2_fast(m - ref) : 1.f;
                        if (grow) m = ref;
                        l *= keep;
                        if (j > 0) {
                            if (!(ok = wait_warp(b_o + my * 8, (done + j - 1) & 1, fail))) break;
                            fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t y[16];
                                tmem_ld16(to + c, y);
                                wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * keep);
                                tmem_st16(to + c, y);
                            }
                        }
                    }
                    // a NaN or infinite score leaves the row's sum NaN, whatever its P
                    if (!(top < INFINITY)) l = NAN;
                    const float base = m == -INFINITY ? 0.f : m;
                    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(-base, -base);
                    uint64_t s0 = pair(0.f, 0.f), s1 = s0;
#pragma unroll
                    for (int c = 0; c < kTile; c += 32) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 w = both(fma2(pair(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), scale2, base2));
                            w = make_float2(exp2_fast(w.x), exp2_fast(w.y));
                            if (e & 1) s1 = add2(s1, pair(w.x, w.y));
                            else s0 = add2(s0, pair(w.x, w.y));
                            pk[e] = pack2<T>(w.x, w.y);
                        }
                        tmem_st16(ts + c / 2, pk);
                        if (c == kFirst - 32) {
                            wait_st();
                            fence_before();
                            arrive(b_ph + my * 8);
                        }
                    }
                    const float2 sum = both(add2(s0, s1));
                    l += sum.x + sum.y;
                    wait_st();
                } else {
                    arrive(b_ph + my * 8);
                }
                fence_before();
                arrive(b_p + my * 8);
            }
            if (ok && steps > 0) ok = wait_warp(b_o + my * 8, (done + steps - 1) & 1, fail);
            fence_after();
            // ---- the rows' results
            if (!ok) l = NAN;  // loud: a wait that ran out leaves no number
            const int f = row0 + row, t = first + f / p.group, qh = h * p.group + f % p.group;
            const int64_t at = (int64_t)t * p.q_heads + qh, pat = (int64_t)g.part * p.tokens * p.q_heads + at;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float odd = 0.f;  // NaN once an element of the row's sum is not finite
            if (rows_here) {
                // The tile's queries are done with: a warp turns its 32 rows round in their place, so
                // that stores run along the rows.  A pass: D 16-bit results or D / 2 32-bit sums.
                unsigned char* area = smem + my * C::kBlock + quarter * (C::kBlock / 4);
                char* to_row = p.direct ? static_cast<char*>(p.out) + (t * p.o_tok + qh * p.o_head) * 2
                                        : reinterpret_cast<char*>(p.part_o + pat * D);
                if (row >= nrows || (!p.direct && l == 0.f)) to_row = nullptr;
                const int passes = p.direct ? 1 : 2;
#pragma unroll 1
                for (int pass = 0; pass < passes; ++pass) {
                    const int cols = D / passes;
#pragma unroll 1
                    for (int c = 0; c < cols; c += 32) {
                        uint32_t y[32];
                        if (steps > 0) {
                            tmem_ld32(to + pass * cols + c, y);
                            wait_ld();
                        }
                        float o0 = 0.f, o1 = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            o0 = fmaf(__uint_as_float(y[e]), 0.f, o0);
                            o1 = fmaf(__uint_as_float(y[e + 1]), 0.f, o1);
                        }
                        odd += o0 + o1;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (l == 0.f) y[e] = 0;
                        if (p.direct) {
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                y[e] = pack2<T>(__uint_as_float(y[2 * e]) * inv, __uint_as_float(y[2 * e + 1]) * inv);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (e < 4 || !p.direct)
                                *reinterpret_cast<uint4*>(area + lane * D * 2 +
                                                          ((((p.direct ? c / 8 : c / 4) + e) ^ lane) & (CH - 1)) * 16) =
                                    make_uint4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        const int r = (i * 32 + lane) / CH, c = lane % CH;
                        char* dst = reinterpret_cast<char*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(to_row), r));
                        const uint4 v = *reinterpret_cast<const uint4*>(area + r * D * 2 + ((c ^ r) & (CH - 1)) * 16);
                        if (dst) *reinterpret_cast<uint4*>(dst + pass * D * 2 + c * 16) = v;
                    }
                    __syncwarp();
                }
                // A value that a row does not see, of a tile that it sees in part, reaches it as 0
                // times the value: where that is NaN, the row is done again alone.
                const bool again = row < nrows && seen < k1 && steps > 0 && odd != odd;
                if (row < nrows && !again) {
                    if (!p.direct) p.part_ml[pat] = make_float2(m, l);
                    else if (p.lse) p.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
                }
                if (__any_sync(kFull, again)) {
                    for (int i = 0; i < 32; ++i) {
                        const int r = __shfl_sync(kFull, row, i), n = __shfl_sync(kFull, seen, i);
                        if (__shfl_sync(kFull, again, i)) row_alone<T, D>(p, g, r, n);
                    }
                }
            }
            fence_before();
            done += steps;
            // the tile's memory and TMEM may be written again
            asm volatile("bar.sync %0, 128;" ::"r"(1 + my) : "memory");
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        tmem_free(tmem, kCols);
    }
}

// ------------------------------------------------------------------ host
template <typename T, int D>
int tc_launch(const AttnParams& p, int ctas, bool pdl, cudaStream_t st) {
    using C = TcCfg<D>;
    static_assert(C::kSmem <= 227 * 1024 && sizeof(TcShared) <= 2048, "shared memory of a CTA");
    const int box = std::gcd(p.page_size, kTile);
    CUtensorMap kmap, vmap;
    int rc = cache_maps(p, std::is_same<T, __half>::value, D, box, &kmap, &vmap);
    auto kernel = p.fill ? attn_tc_kernel<T, D, true> : attn_tc_kernel<T, D, false>;
    static SmemOnce once[2];
    if (rc == TG_OK)
        rc = once[p.fill].raise(reinterpret_cast<const void*>(kernel), C::kSmem);
    if (rc != TG_OK) return rc;
    const dim3 grid((unsigned)ctas);
    if (pdl) return launch_pdl("attn_tc_kernel", kernel, grid, kThreads, C::kSmem, st, p, box, kmap, vmap);
    kernel<<<grid, kThreads, C::kSmem, st>>>(p, box, kmap, vmap);
    return check_launch("attn_tc_kernel");
}

}  // namespace

template <typename T>
int attn_tc_run(const AttnParams& p, int dim, int ctas, bool pdl, cudaStream_t st) {
    return dim == 64 ? tc_launch<T, 64>(p, ctas, pdl, st) : tc_launch<T, 128>(p, ctas, pdl, st);
}
template int attn_tc_run<__half>(const AttnParams&, int, int, bool, cudaStream_t);
template int attn_tc_run<__nv_bfloat16>(const AttnParams&, int, int, bool, cudaStream_t);

}  // namespace tg
