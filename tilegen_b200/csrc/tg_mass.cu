// The attention weight that each cached key gathers (tg_attention_mass_*):
//   mass[key] = decay mass[key] + sum over the rows r that see it of exp(scale q_r k - lse_r),
// the rows being the new tokens of the key's sequence times the query heads of its key head.
//
// A step is S^T = K Q^T of 128 keys and up to 128 rows (tcgen05): the keys lie along the lanes of TMEM,
// so a thread has one key, its sum over the rows crosses no lanes, and a key that is NaN or lies behind
// the sequence stays its own affair.  Four warpgroups make exponentials and sums of a buffer each, so
// that the tensor core works for one while the others keep the special-function units busy.  Sums are
// 32-bit and in a fixed order: calls are bit identical.
//
//   TMEM columns   [128 g, 128 g + 128) S^T of warpgroup g
//   warps 0-15     exponentials and sums, every fourth tile of keys a warpgroup
//   warp 16        fetches tiles of keys by TMA, in boxes of as many rows as divide both a page and a tile
//   warp 17        issues the matrix instructions
//   warp 18        fetches queries by TMA (a box of tokens times heads), and for each row its lse and how
//                  many keys it sees
//   warp 19        looks up the pages of the next unit's keys (and adds up the warpgroups' sums of a unit
//                  with many rows)
//
// * Up to 256 rows of a key head (decoding; the last tokens of a prompt): bound by the keys' bytes.  The
//   rows stay in shared memory, the keys pass through a ring (stream_kernel).  64 sequences of 200 to 4000
//   keys, one token each (284 MB): 56 us, 5.1 TB/s; windows of 32 tokens over 212 MB of keys 48 to 57 us,
//   where the special-function units are 61 % busy too: a warpgroup gives its buffer back only after
//   its exponentials, so that neither unit has work all the time.
// * More rows: bound by the exponentials, 16 a cycle and SM, and the hand-over of buffers between the tensor
//   core and the warpgroups: whole prompts of 300 to 3500 tokens (191 GFLOP that count, 745 million
//   exponentials) 304 us, special-function units 69 % and tensor pipe 35 % active; with exponentials
//   replaced by a product it took 292 us of then 320.  A chunk of 512 keys stays, the rows pass
//   through a ring (rows_kernel), and a thread's sums stay in registers until all rows have passed.  The
//   steps go round the warpgroups, so that under the causal mask, where rows see one to four of the
//   chunk's tiles, none is idle.
//
// CTAs are persistent; a unit of work is (chunk of keys, part of the row tiles) of a (sequence, key
// head).  Each CTA counts the units of all sequences at its begin and takes every gridDim.x-th, so that
// ragged lengths and the causal mask leave no holes in the shares.
#include <algorithm>
#include <cstdlib>
#include <numeric>

#include "tg_tcgen05.cuh"

namespace tg {
namespace {

constexpr int kTile = 128;      // keys of a step
constexpr int kHalfRows = 128;  // rows of a buffer in TMEM
constexpr int kMostRows = 256;  // rows of a key head that stay in shared memory
constexpr int kGroups = 4;      // warpgroups that sum
constexpr int kThreads = kGroups * 128 + 128;
constexpr int kKeysWarp = kGroups * 4, kMmaWarp = kKeysWarp + 1, kRowsWarp = kKeysWarp + 2, kPagesWarp = kKeysWarp + 3;
constexpr uint32_t kCols = 512;
constexpr int kStagesMax = 8;
constexpr int kChunkMax = 8;   // most tiles of a chunk of keys that passes
constexpr int kRowsChunk = 4;  // and of one that stays
constexpr int kSeqs = 512;    // sequences of a launch

struct MassParams : AttnParams {
    const float* row_lse;
    float* mass;
    int64_t m_page, m_slot, m_head;
    float decay;
    // rows: tiles of tile_tokens tokens and tile_heads query heads, head_tiles of them side by side
    int tile_tokens, tile_heads, head_tiles, tile_rows;  // tile_rows: columns of the instructions, a multiple of 16
    int per_head;                                        // 2^16 / tile_heads, rounded up: divides numbers below 256
    int stream;                                          // stream_kernel: one row tile
    int chunk, chunks, splits, split_tiles;              // tiles of keys of a chunk; row tiles of a part
    int box, box_shift;                                  // keys of a box, their log2
    int q_bufs, stages;
    int first_seq, seqs;  // of this launch
    uint64_t wait_ns;     // how long warps wait for one another; 0: as if a wait had run out in every CTA
    float* part;          // with splits > 1: [split][chunk][sequence][key head][key of the chunk]
};

struct MassShared {
    uint64_t q_full[4], q_empty[4], i_full[2], i_empty[2], p_full[2], p_empty[2], a_full, a_empty, full[kStagesMax], empty[kStagesMax], s_full[4],
        s_empty[4], drained;
    uint32_t tmem;
    int fail;
    int passed;                                        // row tiles that have been fetched
    int fewest[2], rows[2];                            // keys that every row of the tile sees; rows
    __align__(16) float lse2[2][kMostRows];            // -lse * log2 e
    __align__(16) int seen[2][kMostRows];              // keys that a row sees, 0 for what is no row
    float acc[kGroups][kRowsChunk * kTile];            // rows_kernel: the sums of each warpgroup at a unit's end
    int page[2][kChunkMax * kTile];                    // pages of a unit's boxes, -1: not in the cache
    int64_t page0[kSeqs];
    int first[kSeqs], n[kSeqs], len[kSeqs];
    int before[kSeqs + 1];  // units of the sequences before
};
constexpr int kSmem = 226 * 1024;
constexpr int kTiles = kSmem - ((int)sizeof(MassShared) + 1023) / 1024 * 1024;  // of them for queries and keys
static_assert(kTiles >= 192 * 1024, "a chunk of keys and two row tiles");

struct Unit {
    Sequence s;
    int b, h, k0, keys, q0, q1, tiles;  // keys k0 .. k0 + keys, row tiles q0 .. q1, tiles of keys
    int split, c;
};

__device__ __forceinline__ int row_tiles(const MassParams& p, const Sequence& s) {
    return (s.asked + p.tile_tokens - 1) / p.tile_tokens * p.head_tiles;
}
// Tiles of the unit's keys that a row of row tile qi may see.
__device__ __forceinline__ int steps_of(const MassParams& p, const Unit& u, int qi) {
    if (!p.causal) return u.tiles;
    const int last = min(((p.head_tiles == 1 ? qi : qi / p.head_tiles) + 1) * p.tile_tokens, u.s.asked) - 1;
    const int64_t seen = (int64_t)u.s.len - u.s.n + last + 1 - u.k0;
    return seen <= 0 ? 0 : ((int)min(seen, (int64_t)u.keys) + kTile - 1) / kTile;
}
// Parts of a sequence's row tiles, and the first of them that sees keys from k0 on (`all`: none does).
// (Parts have whole tokens: head_tiles is 1.)
__device__ __forceinline__ int splits_of(const MassParams& p, const Sequence& s) {
    return (row_tiles(p, s) + p.split_tiles - 1) / p.split_tiles;
}
__device__ __forceinline__ int first_split(const MassParams& p, const Sequence& s, int k0, int all) {
    if (!p.causal) return 0;
    const int64_t behind = (int64_t)k0 - s.len + s.n;  // token i sees them where i >= behind
    if (behind >= s.asked) return all;
    return behind <= 0 ? 0 : (int)behind / (p.split_tiles * p.tile_tokens);
}
// Units of a sequence and one key head.
__device__ __forceinline__ int units_of(const MassParams& p, const Sequence& s) {
    const int step = p.chunk * kTile;
    if (p.splits == 1) return s.n == 0 && p.decay == 1.f ? 0 : (s.len + step - 1) / step;  // (the old weights stay)
    const int all = splits_of(p, s);
    int units = 0;
    for (int k0 = 0; k0 < s.len; k0 += step) units += all - first_split(p, s, k0, all);
    return units;
}

// Fills the table of the launch's sequences; by all threads.
__device__ __forceinline__ void count_units(const MassParams& p, MassShared& sh) {
    for (int i = threadIdx.x; i < kSeqs; i += kThreads) {
        int units = 0;
        if (i < p.seqs) {
            const Sequence s = sequence(p, p.first_seq + i);
            sh.page0[i] = s.page0, sh.first[i] = s.first, sh.n[i] = s.n, sh.len[i] = s.len;
            units = units_of(p, s) * p.kv_heads;
        }
        sh.before[i + 1] = units;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int kEach = kSeqs / 32;
        int v[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum += v[i] = sh.before[threadIdx.x * kEach + i + 1];
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(kFull, scan, o);
            if ((int)threadIdx.x >= o) scan += x;
        }
        scan -= sum;
        if (threadIdx.x == 0) sh.before[0] = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sh.before[threadIdx.x * kEach + i + 1] = scan += v[i];
    }
}

// The units of a CTA, the same for all its warps.
struct Units {
    int at, turn;  // turn: units so far
    __device__ __forceinline__ Units() : at(blockIdx.x), turn(-1) {}
    __device__ __forceinline__ bool next(const MassParams& p, const MassShared& sh, Unit& u) {
        if (at >= sh.before[kSeqs]) return false;
        ++turn;
        // the sequence: the last one with no more units before it
        const int lane = threadIdx.x & 31;
        constexpr int kEach = kSeqs / 32;
        const int coarse = 31 - __clz(__ballot_sync(kFull, sh.before[lane * kEach] <= at));
        const uint32_t fine = __ballot_sync(kFull, lane < kEach && sh.before[coarse * kEach + (lane & (kEach - 1))] <= at);
        const int i = coarse * kEach + 31 - __clz(fine);
        int x = at - sh.before[i];
        at += gridDim.x;
        u.b = p.first_seq + i;
        u.s.page0 = sh.page0[i], u.s.first = sh.first[i], u.s.n = sh.n[i], u.s.len = sh.len[i];
        u.s.asked = min(u.s.n, p.max_q);
        u.h = x % p.kv_heads;
        x /= p.kv_heads;
        const int step = p.chunk * kTile;
        u.c = x, u.split = 0;
        if (p.splits > 1) {
            const int all = splits_of(p, u.s);
            for (u.c = 0;; ++u.c) {
                const int first = first_split(p, u.s, u.c * step, all);
                if (x < all - first) {
                    u.split = first + x;
                    break;
                }
                x -= all - first;
            }
        }
        u.k0 = u.c * step;
        u.keys = min(u.s.len - u.k0, step);
        u.tiles = (u.keys + kTile - 1) / kTile;
        u.q0 = u.split * p.split_tiles;
        u.q1 = min(u.q0 + p.split_tiles, row_tiles(p, u.s));
        return true;
    }
};

// Where the sums of a unit start among the parts.
__device__ __forceinline__ int64_t part_at(const MassParams& p, const Unit& u) {
    return ((((int64_t)u.split * p.chunks + u.c) * p.rows + u.b) * p.kv_heads + u.h) * (p.chunk * kTile);
}
__device__ __forceinline__ int slot_of(const MassParams& p, int key) {
    return p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
}
// Where key `at` of the unit keeps its weight, by the table of its pages; null where there is no such
// page or key.
__device__ __forceinline__ float* mass_at(const MassParams& p, const Unit& u, const int* pages, int at) {
    if (at >= u.keys) return nullptr;
    const int page = pages[at >> p.box_shift];
    return page < 0 ? nullptr : p.mass + page * p.m_page + slot_of(p, u.k0 + at) * p.m_slot + u.h * p.m_head;
}
// Whether what a key has gathered is kept: not that of the call's own tokens, whose slots hold the
// weights of whoever had them before, and not where decay is 0.
__device__ __forceinline__ bool has_old(const MassParams& p, const Unit& u, int key) {
    return p.decay != 0.f && !(p.causal && key >= u.s.len - u.s.n);
}
__device__ __forceinline__ void put(const MassParams& p, const Unit& u, int key, float* to, float old, float sum) {
    if (to) *to = has_old(p, u, key) ? fmaf(old, p.decay, sum) : sum;
}

// A key's sum over COLS rows of S^T: their -lse * log2 e and the keys that they see.  ALL: each sees the
// key.
template <int COLS, bool ALL>
__device__ __forceinline__ float weigh(const uint32_t (&s)[COLS], const float* lse2, const int* seen, int key, float scale) {
    const float4* l4 = reinterpret_cast<const float4*>(lse2);
    if constexpr (ALL) {
        uint64_t part[2] = {0, 0};
        const uint64_t sc = pair(scale, scale);
#pragma unroll
        for (int e = 0; e < COLS; e += 4) {
            const float4 l = l4[e / 4];
            const float2 x = both(fma2(pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sc, pair(l.x, l.y)));
            const float2 y = both(fma2(pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), sc, pair(l.z, l.w)));
            part[0] = add2(part[0], pair(exp2_fast(x.x), exp2_fast(x.y)));
            part[1] = add2(part[1], pair(exp2_fast(y.x), exp2_fast(y.y)));
        }
        const float2 v = both(add2(part[0], part[1]));
        return v.x + v.y;
    } else {
        const int4* n4 = reinterpret_cast<const int4*>(seen);
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < COLS; e += 4) {
            const float4 l = l4[e / 4];
            const int4 n = n4[e / 4];
            part += key < n.x ? exp2_fast(fmaf(__uint_as_float(s[e]), scale, l.x)) : 0.f;
            part += key < n.y ? exp2_fast(fmaf(__uint_as_float(s[e + 1]), scale, l.y)) : 0.f;
            part += key < n.z ? exp2_fast(fmaf(__uint_as_float(s[e + 2]), scale, l.z)) : 0.f;
            part += key < n.w ? exp2_fast(fmaf(__uint_as_float(s[e + 3]), scale, l.w)) : 0.f;
        }
        return part;
    }
}

__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        "\n\t}" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}


// What the warps of a CTA share: addresses of its memory and barriers.
struct Cta {
    MassShared& sh;
    uint32_t sq, ring, tmem, b_full, b_empty, b_qf, b_qe, b_if, b_ie, b_pf, b_pe, b_sf, b_se;
    int q_half, q_block;  // bytes of 64 columns of a row tile, and of the whole tile
    volatile int* fail;
};

// As wait_warp, for what may take as long as all row tiles of a unit do, which are as many as a sequence has
// tokens: the time starts anew with each of them.
__device__ __forceinline__ bool wait_rows(const MassParams& p, const Cta& c, uint32_t bar, uint32_t parity) {
    bool ok = mbar_try(bar, parity);
    if (!ok) {
        const volatile int* passed = &c.sh.passed;
        uint64_t t0 = globaltimer_ns();
        for (int last = *passed;;) {
            if ((ok = mbar_try(bar, parity)) || *c.fail) break;
            const uint64_t t = globaltimer_ns();
            const int now = *passed;
            if (now != last) {
                last = now, t0 = t;
            } else if (t - t0 > p.wait_ns) {
                *c.fail = 1;
                break;
            }
        }
    }
    return __all_sync(kFull, ok);
}

template <int DIM>
__device__ __forceinline__ Cta enter(const MassParams& p, unsigned char* smem, int page_readers, int warp, int lane) {
    MassShared& sh = *reinterpret_cast<MassShared*>(smem + kTiles);
    Cta c{sh};
    c.q_half = p.tile_rows * 128, c.q_block = c.q_half * (DIM / 64);
    c.sq = smem_addr(smem), c.ring = c.sq + p.q_bufs * c.q_block;
    c.b_full = smem_addr(sh.full), c.b_empty = smem_addr(sh.empty), c.b_qf = smem_addr(sh.q_full), c.b_qe = smem_addr(sh.q_empty);
    c.b_if = smem_addr(sh.i_full), c.b_ie = smem_addr(sh.i_empty), c.b_pf = smem_addr(sh.p_full), c.b_pe = smem_addr(sh.p_empty);
    c.b_sf = smem_addr(sh.s_full), c.b_se = smem_addr(sh.s_empty);
    c.fail = &sh.fail;
    if (warp == kMmaWarp) {
        tmem_alloc(smem_addr(&sh.tmem), kCols);
        if (lane == 0) {
            for (int i = 0; i < kStagesMax; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.i_full[i], 1);
                mbar_init(&sh.i_empty[i], kGroups * 4);
                mbar_init(&sh.p_full[i], 1);
                mbar_init(&sh.p_empty[i], page_readers);
            }
            for (int i = 0; i < 4; ++i) {
                mbar_init(&sh.q_full[i], 1);
                mbar_init(&sh.q_empty[i], 1);
                mbar_init(&sh.s_full[i], 1);
                mbar_init(&sh.s_empty[i], 4);
            }
            mbar_init(&sh.a_full, kGroups * 4);
            mbar_init(&sh.a_empty, 1);
            mbar_init(&sh.drained, 1);
            sh.fail = p.wait_ns == 0;
            sh.passed = 0;
            fence_mbar_init();
        }
    }
    count_units(p, sh);
    fence_before();
    __syncthreads();
    fence_after();
    c.tmem = sh.tmem;
    return c;
}
// A warp whose wait has run out stops: it signals nothing and writes nothing more, so that no other takes a
// buffer or a table of pages for what it is not.  The others stop at their next wait.  Then no number of
// the CTA stands, and all keys of all its units get NaN, which the parts' join and a reader cannot miss.
__device__ __noinline__ void spoil(const MassParams& p, const MassShared& sh) {
    Units units;
    Unit u;
    while (units.next(p, sh, u))
        for (int at = threadIdx.x; at < u.keys; at += kThreads) {
            if (p.splits > 1) {
                p.part[part_at(p, u) + at] = NAN;
                continue;
            }
            int page, slot;
            locate(p, p.indices + u.s.page0, u.k0 + at, page, slot);
            if (page >= 0) p.mass[page * p.m_page + slot * p.m_slot + u.h * p.m_head] = NAN;
        }
}
__device__ __forceinline__ void leave(const MassParams& p, const Cta& c, int warp) {
    __syncwarp();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        tmem_free(c.tmem, kCols);
    }
    if (*c.fail) spoil(p, c.sh);
}

// D (+)= A B of STEPS times 16 elements of one 64-column half, both operands in shared memory; `add`: D
// holds something already.  One election and one pair of descriptors for all of them: the issuing warp
// would otherwise take longer than the products (1070 cycles a step against 600).
template <int STEPS>
__device__ __forceinline__ void mma_half(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    static_assert(STEPS == 2 || STEPS == 4, "steps of a half");
    if constexpr (STEPS == 4) {
        asm volatile(
            "{\n\t.reg .pred p, e, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
            "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
            "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
            "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p, e, t;\n\t.reg .b64 a1, b1;\n\t"
            "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
            "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add)
            : "memory");
    }
}

// S^T of a tile of keys and `rows` rows into a buffer, whose barrier completes with it.
template <typename T, int KSTEPS>
__device__ __forceinline__ void product(const Cta& c, uint32_t k, uint32_t q, int rows, int buf) {
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0 : 1;
    constexpr int kHalf = kTile * 128;
    const uint32_t idesc = 1u << 4 | kType << 7 | kType << 10 | (kTile / 16) << 24 | (uint32_t)(rows / 8) << 17;
    const uint64_t a = operand(k, 16), b = operand(q, 16);
    const uint32_t d = c.tmem + buf * kHalfRows;
#pragma unroll
    for (int half = 0; half < KSTEPS / 4; ++half)
        mma_half<4>(d, a + half * (kHalf / 16), b + half * (c.q_half / 16), idesc, half > 0);
    if constexpr (KSTEPS % 4 != 0)
        mma_half<KSTEPS % 4>(d, a + KSTEPS / 4 * (kHalf / 16), b + KSTEPS / 4 * (c.q_half / 16), idesc, 1);
    commit(c.b_sf + buf * 8);
}

// Warp 19: the pages of a unit's boxes.
__device__ __forceinline__ bool find_pages(const MassParams& p, const Cta& c, const Unit& u, int turn, int lane) {
    const int buf = turn & 1;
    if (turn >= 2 && !wait_warp(c.b_pe + buf * 8, (turn / 2 - 1) & 1, c.fail, p.wait_ns)) return false;
    const int64_t* list = p.indices + u.s.page0;
    for (int i = lane; i << p.box_shift < u.keys; i += 32) {
        int page, slot;
        locate(p, list, u.k0 + (i << p.box_shift), page, slot);
        c.sh.page[buf][i] = page;
    }
    __syncwarp();
    if (lane == 0) arrive(c.b_pf + buf * 8);
    return true;
}

// A tile of keys from the unit's key `at` on into shared memory.  A box past the end is not fetched; a page
// that does not exist is fetched from behind the last one, which reads as zeros.
template <int DIM>
__device__ __forceinline__ void fetch_keys(const MassParams& p, const Cta& c, const Unit& u, const int* pages, int at, uint32_t dst,
                                           uint64_t* land, const CUtensorMap* map, int lane) {
    const int boxes = (min(kTile, u.keys - at) + p.box - 1) >> p.box_shift;
    if (lane == 0) mbar_arrive_expect_tx(land, boxes * p.box * DIM * 2);
    __syncwarp();
    for (int b = 0; b < boxes; b += 32) {
        const int i = min(b + lane, boxes - 1), key = at + (i << p.box_shift);
        int page = pages[key >> p.box_shift];
        if (page < 0) page = p.pages;
        const int slot = slot_of(p, u.k0 + key);
        for (int j = 0; j < min(boxes - b, 32); ++j) {
            const int pg = __shfl_sync(kFull, page, j), sl = __shfl_sync(kFull, slot, j);
#pragma unroll
            for (int half = 0; half < DIM / 64; ++half)
                load_box(dst + half * (kTile * 128) + ((b + j) << p.box_shift) * 128, map, half * 64, sl, u.h, pg, smem_addr(land));
        }
    }
}

// Warp 18: row tile qi of the unit into its buffer, and of its rows what the exponentials take.  What is
// read for them is under way while the buffers are waited for: the steps of a tile take less than that.
template <int DIM>
__device__ __forceinline__ bool fetch_rows(const MassParams& p, const Cta& c, const Unit& u, int qi, int nq, const CUtensorMap* map, int lane) {
    constexpr int kEach = kMostRows / 32;
    const int qb = nq % p.q_bufs, ib = nq & 1;
    const int tile = p.head_tiles == 1 ? qi : qi / p.head_tiles, t0 = tile * p.tile_tokens, h0 = (qi - tile * p.head_tiles) * p.tile_heads;
    const int rows = min(p.tile_tokens, u.s.asked - t0) * p.tile_heads;
    const float* lse = p.row_lse + (int64_t)(u.s.first + t0) * p.q_heads + u.h * p.group + h0;
    float l[kEach];
    int seen[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int r = lane + k * 32, i = r * p.per_head >> 16, x = r - i * p.tile_heads;  // token and head of the tile
        const bool there = r < rows && h0 + x < p.group;
        l[k] = 0.f;
        seen[k] = 0;
        if (there) {
            l[k] = __ldg(lse + (int64_t)i * p.q_heads + x);
            seen[k] = keys_seen(p, u.s, t0 + i, u.s.len, u.s.len);
        }
    }
    if (nq >= p.q_bufs && !wait_warp(c.b_qe + qb * 8, (nq / p.q_bufs - 1) & 1, c.fail, p.wait_ns)) return false;
    if (lane == 0) mbar_arrive_expect_tx(&c.sh.q_full[qb], p.tile_tokens * p.tile_heads * DIM * 2);
    __syncwarp();
#pragma unroll
    for (int half = 0; half < DIM / 64; ++half)
        load_box3(c.sq + qb * c.q_block + half * c.q_half, map, half * 64, u.h * p.group + h0, u.s.first + t0, c.b_qf + qb * 8);
    if (nq >= 2 && !wait_warp(c.b_ie + ib * 8, (nq / 2 - 1) & 1, c.fail, p.wait_ns)) return false;
    int fewest = INT_MAX;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int r = lane + k * 32;
        if (k * 32 >= rows) break;
        l[k] *= -1.4426950408889634f;
        if (l[k] == INFINITY) seen[k] = 0;
        c.sh.lse2[ib][r] = l[k];
        c.sh.seen[ib][r] = seen[k];
        if (r < rows) fewest = min(fewest, seen[k]);
    }
    fewest = __reduce_min_sync(kFull, fewest);
    if (lane == 0) {
        c.sh.fewest[ib] = fewest;
        c.sh.rows[ib] = rows;
    }
    __syncwarp();
    if (lane == 0) {
        *static_cast<volatile int*>(&c.sh.passed) = nq + 1;
        arrive(c.b_if + ib * 8);
    }
    return true;
}
// Leaves no copy of rows under way.
__device__ __forceinline__ void drain_rows(const MassParams& p, const Cta& c, int nq) {
    __syncwarp();
    if (*c.fail)
        for (int i = max(0, nq - p.q_bufs); i <= nq; ++i) mbar_wait_brief(&c.sh.q_full[i % p.q_bufs], i / p.q_bufs & 1);
}

// A key's sum over the rows [row0, row0 + cols) of row tile ib, whose S^T is in TMEM at t.
__device__ __forceinline__ float sum_rows(const MassParams& p, const Cta& c, uint32_t t, int ib, int row0, int cols, int key, bool all) {
    const float* lse2 = &c.sh.lse2[ib][row0];
    const int* seen = &c.sh.seen[ib][row0];
    const int lane = threadIdx.x & 31;
    float sum = 0.f;
    if (p.tile_rows <= 16) {
        uint32_t s[16];
        tmem_ld16(t, s);
        wait_ld();
        return weigh<16, false>(s, lse2, seen, key, p.scale_log2);
    }
    if (cols <= 0) return 0.f;
#pragma unroll 1
    for (int x = 0; x < cols; x += 32) {
        uint32_t s[32];
        tmem_ld32(t + x, s);
        wait_ld();
        if (all && x + 32 <= cols) sum += weigh<32, true>(s, lse2 + x, seen + x, key, p.scale_log2);
        else if (__reduce_max_sync(kFull, seen[x + lane]) > key - lane)  // one of the 32 rows sees one of the warp's keys
            sum += weigh<32, false>(s, lse2 + x, seen + x, key, p.scale_log2);
    }
    return sum;
}

// One row tile: DIM is the head size rounded up to 64 elements, KSTEPS its steps of 16.
template <typename T, int DIM, int KSTEPS>
__global__ void __launch_bounds__(kThreads, 1) stream_kernel(const __grid_constant__ MassParams p,
                                                             const __grid_constant__ CUtensorMap kmap,
                                                             const __grid_constant__ CUtensorMap qmap) {
    constexpr int kBlock = kTile * DIM * 2;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    const Cta c = enter<DIM>(p, smem, kGroups * 4 + 1, warp, lane);
    const int halves = p.tile_rows > kHalfRows ? 2 : 1;
    Units units;
    Unit u;
    bool ok = true;

    if (warp == kMmaWarp) {
        int f = 0, nq = 0;  // tiles of keys and row tiles so far
        while (ok && units.next(p, c.sh, u)) {
            if (u.s.asked == 0) continue;
            const int qb = nq % p.q_bufs;
            ok = wait_warp(c.b_qf + qb * 8, nq / p.q_bufs & 1, c.fail, p.wait_ns);
            for (int j = 0; ok && j < u.tiles; ++j, ++f) {
                const int st = f % p.stages, buf = f % kGroups;
                ok = wait_warp(c.b_full + st * 8, f / p.stages & 1, c.fail, p.wait_ns);
                for (int half = 0; ok && half < halves; ++half) {
                    const int i = f / kGroups * halves + half;
                    ok = i < 1 || wait_warp(c.b_se + buf * 8, (i - 1) & 1, c.fail, p.wait_ns);
                    if (!ok) break;
                    fence_after();
                    product<T, KSTEPS>(c, c.ring + st * kBlock, c.sq + qb * c.q_block + half * kHalfRows * 128,
                                       half ? p.tile_rows - kHalfRows : min(p.tile_rows, kHalfRows), buf);
                }
                if (!ok) break;
                commit(c.b_empty + st * 8);
            }
            if (ok) commit(c.b_qe + qb * 8);
            ++nq;
        }
        if (!ok || *c.fail) {  // leave no product under way
            commit(smem_addr(&c.sh.drained));
            mbar_wait(&c.sh.drained, 0);
        }
    } else if (warp == kKeysWarp) {
        int f = 0;
        while (ok && units.next(p, c.sh, u)) {
            const int buf = units.turn & 1;
            ok = wait_warp(c.b_pf + buf * 8, units.turn / 2 & 1, c.fail, p.wait_ns);
            for (int j = 0; ok && u.s.asked > 0 && j < u.tiles; ++j, ++f) {
                const int st = f % p.stages;
                if (f >= p.stages && !(ok = wait_warp(c.b_empty + st * 8, (f / p.stages - 1) & 1, c.fail, p.wait_ns))) break;
                fetch_keys<DIM>(p, c, u, c.sh.page[buf], j * kTile, c.ring + st * kBlock, &c.sh.full[st], &kmap, lane);
            }
            __syncwarp();
            if (ok && lane == 0) arrive(c.b_pe + buf * 8);
        }
        __syncwarp();
        if (*c.fail)  // leave no copy under way
            for (int i = max(0, f - p.stages); i < f + p.stages; ++i)
                mbar_wait_brief(&c.sh.full[i % p.stages], i / p.stages & 1);
    } else if (warp == kRowsWarp) {
        int nq = 0;
        while (ok && units.next(p, c.sh, u)) {
            if (u.s.asked == 0) continue;
            ok = fetch_rows<DIM>(p, c, u, 0, nq, &qmap, lane);
            if (ok) ++nq;
        }
        drain_rows(p, c, nq);
    } else if (warp == kPagesWarp) {
        while (ok && units.next(p, c.sh, u)) ok = find_pages(p, c, u, units.turn, lane);
    } else {
        const int my = warp >> 2, key_of = tid & (kTile - 1);
        const uint32_t ts = c.tmem + my * kHalfRows + ((uint32_t)(warp & 3) << 21);
        int f = 0, nq = 0;
        while (ok && units.next(p, c.sh, u)) {
            const int pb = units.turn & 1, ib = nq & 1, f0 = f, tiles = u.s.asked > 0 ? u.tiles : 0;
            ok = wait_warp(c.b_pf + pb * 8, units.turn / 2 & 1, c.fail, p.wait_ns);
            const int* pages = c.sh.page[pb];
            auto old_of = [&](int at, float*& to, float& old) {
                to = mass_at(p, u, pages, at), old = 0.f;
                if (to && has_old(p, u, u.k0 + at)) old = *to;
            };
            float *to = nullptr, *to_next;
            float old = 0.f, old_next;
            if (tiles > 0) {
                // the old weights of my next tile are under way
                const int skip = (my - f % kGroups + kGroups) % kGroups;
                if (ok) old_of(skip * kTile + key_of, to, old);
                ok = ok && wait_warp(c.b_if + ib * 8, nq / 2 & 1, c.fail, p.wait_ns);
                const int rows = c.sh.rows[ib], fewest = c.sh.fewest[ib];
                for (f += skip; ok && f < f0 + tiles; f += kGroups) {
                    const int at = (f - f0) * kTile + key_of, key = u.k0 + at;
                    old_of(at + kGroups * kTile, to_next, old_next);
                    const bool all = u.k0 + min(at - key_of + kTile, u.keys) <= fewest;  // every row sees every key
                    float sum = 0.f;
                    for (int half = 0; ok && half < halves; ++half) {
                        ok = wait_warp(c.b_sf + my * 8, (f / kGroups * halves + half) & 1, c.fail, p.wait_ns);
                        if (!ok) break;
                        fence_after();
                        sum += sum_rows(p, c, ts, ib, half * kHalfRows, min(rows - half * kHalfRows, kHalfRows), key, all);
                        fence_before();
                        __syncwarp();
                        if (lane == 0) arrive(c.b_se + my * 8);
                    }
                    if (!ok) break;
                    put(p, u, key, to, old, sum);
                    to = to_next, old = old_next;
                }
                f = f0 + tiles;
                __syncwarp();
                if (ok && lane == 0) arrive(c.b_ie + ib * 8);
                ++nq;
            } else if (ok) {  // no row: the old weights decay
                for (int at = tid; at < u.keys; at += kGroups * kTile) {
                    old_of(at, to, old);
                    put(p, u, u.k0 + at, to, old, 0.f);
                }
            }
            __syncwarp();
            if (ok && lane == 0) arrive(c.b_pe + pb * 8);
        }
    }
    leave(p, c, warp);
}

// Many row tiles: a chunk of keys stays in shared memory while they pass.
template <typename T, int DIM, int KSTEPS>
__global__ void __launch_bounds__(kThreads, 1) rows_kernel(const __grid_constant__ MassParams p,
                                                           const __grid_constant__ CUtensorMap kmap,
                                                           const __grid_constant__ CUtensorMap qmap) {
    constexpr int kBlock = kTile * DIM * 2;
    constexpr int kChunk = DIM > 128 ? kRowsChunk / 2 : kRowsChunk;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    const Cta c = enter<DIM>(p, smem, 2, warp, lane);
    Units units;
    Unit u;
    bool ok = true;

    if (warp == kMmaWarp) {
        int nq = 0;             // row tiles so far
        uint32_t used = 0;      // parity of the tiles of keys, by bit
        uint32_t began = 0, emptied = 0;  // buffers that were written, and the parity of their emptying
        while (ok && units.next(p, c.sh, u)) {
            int here = 0, g = 0;  // tiles of keys that have come; steps of the unit
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                const int steps = steps_of(p, u, qi);
                if (steps == 0) continue;
                const int qb = nq % p.q_bufs;
                ok = wait_warp(c.b_qf + qb * 8, nq / p.q_bufs & 1, c.fail, p.wait_ns);
                for (int j = 0; ok && j < steps; ++j, ++g) {
                    if (j >= here) {
                        ok = wait_warp(c.b_full + j * 8, used >> j & 1, c.fail, p.wait_ns);
                        used ^= 1u << j;
                        here = j + 1;
                    }
                    const int buf = g % kGroups;
                    if (began >> buf & 1) {
                        ok = ok && wait_warp(c.b_se + buf * 8, emptied >> buf & 1, c.fail, p.wait_ns);
                        emptied ^= 1u << buf;
                    }
                    began |= 1u << buf;
                    if (!ok) break;
                    fence_after();
                    product<T, KSTEPS>(c, c.ring + j * kBlock, c.sq + qb * c.q_block, p.tile_rows, buf);
                    if (qi == u.q1 - 1) commit(c.b_empty + j * 8);  // the last rows see the most keys
                }
                if (ok) commit(c.b_qe + qb * 8);
                ++nq;
            }
        }
        if (!ok || *c.fail) {  // leave no product under way
            commit(smem_addr(&c.sh.drained));
            mbar_wait(&c.sh.drained, 0);
        }
    } else if (warp == kKeysWarp) {
        uint32_t began = 0, freed = 0;  // whether a place was filled before, and the parity of its emptying
        uint32_t landed = 0;
        while (ok && units.next(p, c.sh, u)) {
            const int buf = units.turn & 1, tiles = u.q1 > u.q0 ? steps_of(p, u, u.q1 - 1) : 0;
            ok = wait_rows(p, c, c.b_pf + buf * 8, units.turn / 2 & 1);
            for (int j = 0; ok && j < tiles; ++j) {
                if (began >> j & 1) {
                    ok = wait_rows(p, c, c.b_empty + j * 8, freed >> j & 1);
                    freed ^= 1u << j;
                }
                if (!ok) break;
                began |= 1u << j;
                landed ^= 1u << j;
                fetch_keys<DIM>(p, c, u, c.sh.page[buf], j * kTile, c.ring + j * kBlock, &c.sh.full[j], &kmap, lane);
            }
            __syncwarp();
            if (ok && lane == 0) arrive(c.b_pe + buf * 8);
        }
        __syncwarp();
        if (*c.fail)  // leave no copy under way
            for (int j = 0; j < p.chunk; ++j)
                if (began >> j & 1) mbar_wait_brief(&c.sh.full[j], (landed >> j & 1) ^ 1);
    } else if (warp == kRowsWarp) {
        int nq = 0;
        while (ok && units.next(p, c.sh, u))
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                if (steps_of(p, u, qi) == 0) continue;
                ok = fetch_rows<DIM>(p, c, u, qi, nq, &qmap, lane);
                if (ok) ++nq;
            }
        drain_rows(p, c, nq);
    } else if (warp == kPagesWarp) {
        // the pages of a unit ahead, and the sums of one that has been made
        Units made;
        Unit v;
        bool more = units.next(p, c.sh, u);
        ok = !more || find_pages(p, c, u, units.turn, lane);
        while (ok && made.next(p, c.sh, v)) {
            more = more && units.next(p, c.sh, u);
            ok = (!more || find_pages(p, c, u, units.turn, lane)) && wait_rows(p, c, smem_addr(&c.sh.a_full), made.turn & 1);
            if (!ok) break;
            const int pb = made.turn & 1;
            for (int at = lane; at < v.keys; at += 32) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kGroups; ++w) sum += c.sh.acc[w][at];
                if (p.splits > 1) {
                    p.part[part_at(p, v) + at] = sum;
                } else {
                    float* const to = mass_at(p, v, c.sh.page[pb], at);
                    put(p, v, v.k0 + at, to, to && has_old(p, v, v.k0 + at) ? *to : 0.f, sum);
                }
            }
            __syncwarp();
            if (lane == 0) {
                arrive(smem_addr(&c.sh.a_empty));
                arrive(c.b_pe + pb * 8);
            }
        }
    } else {
        const int my = warp >> 2, key_of = tid & (kTile - 1);
        const uint32_t ts = c.tmem + my * kHalfRows + ((uint32_t)(warp & 3) << 21);
        int nq = 0, made = 0;
        while (ok && units.next(p, c.sh, u)) {
            float acc[kChunk];
#pragma unroll
            for (int m = 0; m < kChunk; ++m) acc[m] = 0.f;
            int g = 0;  // steps of the unit
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                const int steps = steps_of(p, u, qi);
                if (steps == 0) continue;
                const int ib = nq & 1;
                ok = wait_warp(c.b_if + ib * 8, nq / 2 & 1, c.fail, p.wait_ns);
                const int rows = c.sh.rows[ib], fewest = c.sh.fewest[ib];
                for (int j = (my - g % kGroups + kGroups) % kGroups; ok && j < steps; j += kGroups) {
                    ok = wait_warp(c.b_sf + my * 8, made & 1, c.fail, p.wait_ns);
                    if (!ok) break;
                    fence_after();
                    const int at = j * kTile + key_of;
                    const bool all = u.k0 + min((j + 1) * kTile, u.keys) <= fewest;  // every row sees every key
                    const float sum = sum_rows(p, c, ts, ib, 0, rows, u.k0 + at, all);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(c.b_se + my * 8);
                    ++made;
#pragma unroll
                    for (int m = 0; m < kChunk; ++m) acc[m] += m == j ? sum : 0.f;
                }
                __syncwarp();
                if (ok && lane == 0) arrive(c.b_ie + ib * 8);
                ++nq;
                g += steps;
            }
            ok = ok && (units.turn == 0 || wait_warp(smem_addr(&c.sh.a_empty), (units.turn - 1) & 1, c.fail, p.wait_ns));
            if (!ok) break;
#pragma unroll
            for (int m = 0; m < kChunk; ++m) c.sh.acc[my][m * kTile + key_of] = acc[m];
            __syncwarp();
            if (lane == 0) arrive(smem_addr(&c.sh.a_full));
        }
    }
    leave(p, c, warp);
}

// mass of the keys of a (chunk, sequence, key head) from the parts of its row tiles, in their order.
__global__ void __launch_bounds__(256) mass_join_kernel(const __grid_constant__ MassParams p) {
    pdl_wait();
    Unit u;
    int x = blockIdx.x;
    u.h = x % p.kv_heads, x /= p.kv_heads;
    u.b = x % p.rows, u.c = x / p.rows;
    u.s = sequence(p, u.b);
    u.k0 = u.c * p.chunk * kTile;
    u.keys = min(u.s.len - u.k0, p.chunk * kTile);
    if (u.keys <= 0 || (u.s.n == 0 && p.decay == 1.f)) return;
    const int all = splits_of(p, u.s), first = first_split(p, u.s, u.k0, all);
    for (int at = threadIdx.x; at < u.keys; at += blockDim.x) {
        int page, slot;
        locate(p, p.indices + u.s.page0, u.k0 + at, page, slot);
        if (page < 0) continue;
        float* const to = p.mass + page * p.m_page + slot * p.m_slot + u.h * p.m_head;
        const bool kept = has_old(p, u, u.k0 + at);
        const float old = kept ? *to : 0.f;
        float sum = 0.f;
        for (u.split = first; u.split < all; ++u.split) sum += p.part[part_at(p, u) + at];
        *to = kept ? fmaf(old, p.decay, sum) : sum;
    }
}

// ------------------------------------------------------------------ host
// Units enough that the last ones end together; with the causal mask about half of them have steps.
// Whole prompts of 300 to 3500 tokens: 330 us with 64 an SM, 318 with 128.
constexpr int64_t kManyUnits = kSMs * 128;

// kept: the plan of the most rows that max_q_len allows, whatever the call's tokens.
int make_plan(const tg_attention_mass_args* a, MassParams* out, const char* op, bool kept = false) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_cache(a->cache, op);
    if (rc == TG_OK && !a->pages) rc = set_error(TG_EINVAL, "%s: null page table", op);
    if (rc != TG_OK) return rc;
    const tg_paged_kv& c = *a->cache;
    const tg_csr& t = *a->pages;
    if (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 256)
        return set_error(TG_EUNSUPPORTED, "%s: head dim must be 64, 96, 128 or 256 (got %d)", op, c.dim);
    if (a->q_heads < 1 || a->q_heads % c.heads)
        return set_error(TG_EINVAL, "%s: q_heads (%d) must be a multiple of the cache's heads (%d)", op, a->q_heads, c.heads);
    if (a->tokens < 0 || a->tokens > INT32_MAX || t.rows < 0 || t.rows > INT32_MAX || t.nnz < 0)
        return set_error(TG_EINVAL, "%s: bad size (tokens=%lld sequences=%lld pages=%lld)", op, (long long)a->tokens,
                         (long long)t.rows, (long long)t.nnz);
    if (a->max_seq_len < 0 || a->max_q_len < 0) return set_error(TG_EINVAL, "%s: negative max_seq_len or max_q_len", op);
    if (a->q_indptr && a->tokens > 0 && a->max_q_len == 0)
        return set_error(TG_EINVAL, "%s: a max_q_len of 0 weighs none of the %lld tokens", op, (long long)a->tokens);
    if (!(a->scale > 0.0) || a->scale > 1e30) return set_error(TG_EINVAL, "%s: scale must be positive", op);
    if (!(a->decay >= 0.0) || a->decay > 1e30) return set_error(TG_EINVAL, "%s: decay must be finite and not negative", op);
    if (a->flags & ~(TG_FLAG_CAUSAL | TG_FLAG_BOUNDS_CHECK)) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    const int64_t slots = c.pages == 0 ? 0 : t.nnz > INT32_MAX / c.page_size ? INT32_MAX / 2 : t.nnz * c.page_size;
    const int64_t max_seq = std::min({a->max_seq_len, slots, (int64_t)INT32_MAX / 2});
    const int64_t max_q = kept ? std::min<int64_t>(std::max<int64_t>(a->max_q_len, 1), INT32_MAX)
                          : a->q_indptr ? std::min(a->max_q_len, a->tokens)
                                        : 1;

    MassParams& p = *out;
    p = {};
    p.q = a->q.data, p.k = c.k, p.v = c.k;
    p.q_tok = stride_of(a->tokens, a->q.token_stride), p.q_head = stride_of(a->q_heads, a->q.head_stride);
    p.k_page = p.v_page = stride_of(c.pages, c.k_page_stride);
    p.k_slot = p.v_slot = stride_of(c.page_size, c.k_slot_stride);
    p.k_head = p.v_head = stride_of(c.heads, c.k_head_stride);
    p.pages = (int)c.pages, p.page_size = (int)c.page_size;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (c.page_size == (1ll << i)) p.page_shift = i;
    p.q_heads = a->q_heads, p.kv_heads = c.heads, p.group = a->q_heads / c.heads;
    p.tokens = (int)a->tokens, p.rows = (int)t.rows;
    p.q_indptr = a->q_indptr, p.indptr = t.indptr, p.indices = t.indices, p.seq_len = a->seq_len, p.nnz = t.nnz;
    p.max_seq = (int)max_seq, p.max_q = (int)max_q;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.causal = (a->flags & TG_FLAG_CAUSAL) != 0;
    p.row_lse = a->lse, p.mass = a->mass.data, p.decay = (float)a->decay;
    p.m_page = stride_of(c.pages, a->mass.page_stride), p.m_slot = stride_of(c.page_size, a->mass.slot_stride);
    p.m_head = stride_of(c.heads, a->mass.head_stride);

    p.box = std::gcd(p.page_size, kTile);
    while (1 << p.box_shift < p.box) ++p.box_shift;
    // Row tiles: up to 256 rows of a key head (128 for heads of 256, whose tiles take twice the room) stay in
    // shared memory; of more rows 128 (64) at a time pass.  A tile has whole tokens, or where one token's
    // heads are more than that, a part of its heads.
    const int dim = (c.dim + 63) / 64 * 64, most = dim > 128 ? kMostRows / 2 : kMostRows;
    p.stream = max_q * p.group <= most;
    const int rows = p.stream ? most : most / 2;
    p.tile_heads = std::min(p.group, rows);
    p.head_tiles = (p.group + p.tile_heads - 1) / p.tile_heads;
    p.tile_tokens = (int)std::max<int64_t>(1, std::min<int64_t>(max_q, rows / p.tile_heads));
    p.tile_rows = (p.tile_tokens * p.tile_heads + 15) / 16 * 16;
    p.per_head = (65536 + p.tile_heads - 1) / p.tile_heads;
    const int64_t q_tiles = std::max<int64_t>(1, ceil_div(max_q, p.tile_tokens)) * p.head_tiles, k_tiles = std::max<int64_t>(1, ceil_div(max_seq, kTile));
    const int q_block = p.tile_rows * dim * 2, k_block = kTile * dim * 2;
    const int64_t pairs = std::max<int64_t>(1, t.rows * c.heads);
    if (p.stream) {
        // Chunks as long as leaves six units a CTA: each fetches its rows anew.  One sequence of 60000 keys 31
        // us, 55 with 16 units a CTA; 64 of 200 to 4000 keys 57 and 58 us.
        p.chunk = (int)std::min<int64_t>(kChunkMax, std::max<int64_t>(1, pairs * k_tiles / (kSMs * 6)));
        p.q_bufs = 2 * q_block + 4 * k_block <= kTiles ? 2 : 1;
        p.stages = std::min(kStagesMax, (kTiles - p.q_bufs * q_block) / k_block);
    } else {
        p.chunk = dim > 128 ? kRowsChunk / 2 : kRowsChunk;
        p.q_bufs = std::min(4, (kTiles - p.chunk * k_block) / q_block);
    }
    p.chunks = (int)ceil_div(k_tiles, p.chunk);
    // Where that makes few units the row tiles are shared out too, at least four to a part.
    p.splits = p.head_tiles > 1 ? 1 : (int)std::max<int64_t>(1, std::min(ceil_div(kManyUnits, pairs * p.chunks), q_tiles / 4));
    p.split_tiles = (int)ceil_div(q_tiles, p.splits);
    p.splits = (int)std::max<int64_t>(1, ceil_div(q_tiles, p.split_tiles));
    if (pairs * p.chunks * p.splits > INT32_MAX - kSMs) return set_error(TG_EUNSUPPORTED, "%s: too many sequences for one launch", op);
    return TG_OK;
}

size_t mass_bytes(const MassParams& p) {
    return p.splits > 1 ? (size_t)p.splits * p.chunks * p.rows * p.kv_heads * p.chunk * kTile * sizeof(float) : 0;
}
// Of any smaller call: parts are made only until there are kManyUnits units, of one row of parts less.
size_t mass_enough(const MassParams& p) {
    return p.stream || p.head_tiles > 1 ? 0 : (size_t)(2 * kManyUnits) * p.chunk * kTile * sizeof(float);
}

// Whole milliseconds from TG_MASS_WAIT_MS in the environment, a minute at most; else two seconds, where the
// waits are microseconds.
uint64_t wait_limit() {
    static const uint64_t ns = [] {
        const char* text = std::getenv("TG_MASS_WAIT_MS");
        char* end = nullptr;
        const long ms = text ? std::strtol(text, &end, 10) : 0;
        return !text || end == text || *end || ms < 0 ? kWaitNs : (uint64_t)std::min(ms, 60000l) * 1000000;
    }();
    return ns;
}

template <typename T, int DIM, int KSTEPS>
int mass_run(const MassParams& p, const CUtensorMap& kmap, const CUtensorMap& qmap, cudaStream_t st) {
    auto kernel = p.stream ? stream_kernel<T, DIM, KSTEPS> : rows_kernel<T, DIM, KSTEPS>;
    static SmemOnce once[2];
    int rc = once[p.stream].raise(reinterpret_cast<const void*>(kernel), kSmem);
    if (rc != TG_OK) return rc;
    MassParams some = p;
    for (some.first_seq = 0; some.first_seq < p.rows; some.first_seq += kSeqs) {
        some.seqs = std::min(kSeqs, p.rows - some.first_seq);
        const int grid = (int)std::min<int64_t>((int64_t)some.seqs * p.kv_heads * p.chunks * p.splits, kSMs);
        kernel<<<(unsigned)grid, kThreads, kSmem, st>>>(some, kmap, qmap);
        rc = check_launch("attention_mass kernel");
        if (rc != TG_OK) return rc;
    }
    if (p.splits == 1) return TG_OK;
    return launch_pdl("mass_join_kernel", mass_join_kernel, dim3((unsigned)(p.rows * p.kv_heads * p.chunks)), 256, 0, st, p);
}

template <typename T>
int attention_mass(const tg_attention_mass_args* a, void* ws, size_t ws_bytes, tg_stream_t stream, const char* op) {
    MassParams p;
    int rc = make_plan(a, &p, op);
    if (rc == TG_OK) rc = check_table(a->pages, a->cache, a->tokens, a->q_indptr, a->seq_len, op);
    if (rc != TG_OK) return rc;
    const tg_paged_kv& c = *a->cache;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.rows == 0 || p.max_seq == 0) return TG_OK;
    if (!a->seq_len || !a->pages->indptr) return set_error(TG_EINVAL, "%s: null indptr/seq_len", op);
    if (!a->mass.data) return set_error(TG_EINVAL, "%s: null mass", op);
    if (a->tokens > 0 && (!a->q.data || !a->lse)) return set_error(TG_EINVAL, "%s: null q/lse", op);
    if (a->flags & TG_FLAG_BOUNDS_CHECK) {
        rc = paged_bounds_check(*a->pages, c.page_size, a->seq_len, a->max_seq_len, a->tokens, a->q_indptr,
                                a->q_indptr ? a->max_q_len : 1, nullptr, 0, false, op, st);
        if (rc != TG_OK) return rc;
    }
    const uint64_t at = reinterpret_cast<uint64_t>(p.q) | reinterpret_cast<uint64_t>(p.k);
    const uint64_t strides = (uint64_t)(p.q_tok | p.q_head | p.k_page | p.k_slot | p.k_head);
    if (at % 16 || strides % 8)
        return set_error(TG_EINVAL, "%s: rows must be 16-byte aligned (strides multiples of 8 elements)", op);
    const size_t need = mass_bytes(p);
    if (ws_bytes < need || (need && !ws)) return set_error(TG_ENOMEM, "%s: workspace of %zu bytes needed (got %zu)", op, need, ws_bytes);
    if (reinterpret_cast<uintptr_t>(ws) % 16) return set_error(TG_EINVAL, "%s: the workspace must be 16-byte aligned", op);
    p.part = static_cast<float*>(ws);
    p.wait_ns = wait_limit();
    constexpr bool kIsHalf = std::is_same<T, __half>::value;
    CUtensorMap kmap, vmap, qmap;
    rc = cache_maps(p, kIsHalf, c.dim, p.box, &kmap, &vmap);
    if (rc == TG_OK) rc = rows_map(p, kIsHalf, c.dim, p.tile_heads, p.tile_tokens, &qmap);
    if (rc != TG_OK) return rc;
    switch (c.dim) {
        case 64: return mass_run<T, 64, 4>(p, kmap, qmap, st);
        case 96: return mass_run<T, 128, 6>(p, kmap, qmap, st);
        case 128: return mass_run<T, 128, 8>(p, kmap, qmap, st);
        default: return mass_run<T, 256, 16>(p, kmap, qmap, st);
    }
}

}  // namespace
}  // namespace tg

extern "C" {

size_t tg_attention_mass_workspace_bytes(const tg_attention_mass_args* a) {
    tg::MassParams p;
    return tg::make_plan(a, &p, "tg_attention_mass", true) == TG_OK ? tg::mass_enough(p) : 0;
}

size_t tg_attention_mass_needed_bytes(const tg_attention_mass_args* a) {
    tg::MassParams p;
    return tg::make_plan(a, &p, "tg_attention_mass") == TG_OK ? tg::mass_bytes(p) : 0;
}

int tg_attention_mass_f16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::attention_mass<__half>(a, workspace, workspace_bytes, stream, "tg_attention_mass_f16");
}

int tg_attention_mass_bf16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::attention_mass<__nv_bfloat16>(a, workspace, workspace_bytes, stream, "tg_attention_mass_bf16");
}

}  // extern "C"
