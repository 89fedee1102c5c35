// The attention weight that each cached key gathers (tg_attention_mass_*):
//   mass[key] = decay mass[key] + sum over the rows r that see it of exp(scale q_r k - lse_r),
// the rows being the new tokens of the key's sequence times the query heads of its key head.
//
// A step is S^T = K Q^T of 128 keys and up to 256 rows: the keys lie along the lanes of TMEM, so a
// thread has one key, its sum over the rows crosses no lanes, and a key that is NaN or lies behind the
// sequence stays its own affair.  Two warpgroups take turns, so that one's exponentials run while the
// tensor core works for the other.
//
//   TMEM columns      [0,256) S^T of warpgroup 0    [256,512) of warpgroup 1
//   warps 0-3, 4-7    exponentials and sums of every other step
//   warp 8            fetches tiles of keys into a ring of shared memory by TMA, in boxes of as many
//                     rows as divide both a page and a tile
//   warp 9            issues the matrix instructions
//   warp 10           fetches queries by TMA (a box of tokens times heads), and for each row its lse
//                     and how many keys it sees
//
// CTAs are persistent; a unit of work is (part of the row tiles, chunk of keys, sequence, key head).
// A unit with one row tile (decoding; the last tokens of a prompt) writes its sums as they come, the
// others keep them in shared memory, one place for each thread, until all row tiles are done.  Sums
// are 32-bit, in a fixed order: calls are bit identical.
#include <algorithm>
#include <numeric>

#include "tg_tcgen05.cuh"

namespace tg {
namespace {

constexpr int kTile = 128;      // keys of a step
constexpr int kMostRows = 256;  // rows of a row tile: columns of an instruction
constexpr int kThreads = 384;
constexpr uint32_t kCols = 512;
constexpr int kStagesMax = 8;
constexpr int kChunkMax = 8;  // most tiles of a chunk of keys

struct MassParams : AttnParams {
    const float* row_lse;
    float* mass;
    int64_t m_page, m_slot, m_head;
    float decay;
    // rows: tiles of tile_tokens tokens and tile_heads query heads, head_tiles of them side by side
    int tile_tokens, tile_heads, head_tiles, tile_rows;  // tile_rows: columns of the instructions, a multiple of 16
    int chunk, chunks, splits, split_tiles;              // tiles of keys of a chunk; row tiles of a part
    int units, q_bufs, stages;
    float* part;  // with splits > 1: [split][chunk][sequence][key head][key of the chunk]
};

struct MassShared {
    uint64_t q_full[2], q_empty[2], i_full[2], i_empty[2], full[kStagesMax], empty[kStagesMax], s_full[2], s_empty[2], drained;
    uint32_t tmem;
    int fail;
    int fewest[2], rows[2];          // keys that every row of the tile sees; rows
    float lse2[2][kMostRows];        // lse * log2 e
    int seen[2][kMostRows];          // keys that a row sees, 0 for what is no row
    float acc[2][kChunkMax * kTile];  // [warpgroup][key of the chunk]
};

constexpr int kSmem = 226 * 1024;
constexpr int kTiles = kSmem - ((int)sizeof(MassShared) + 1023) / 1024 * 1024;  // of them for queries and keys

struct Unit {
    Sequence s;
    int h, k0, keys, q0, q1, tiles;  // keys k0 .. k0 + keys, row tiles q0 .. q1, tiles of keys
    int id;
};

__device__ __forceinline__ int row_tiles(const MassParams& p, const Sequence& s) {
    return (s.asked + p.tile_tokens - 1) / p.tile_tokens * p.head_tiles;
}
// Tiles of the unit's keys that a row of row tile qi may see.
__device__ __forceinline__ int steps_of(const MassParams& p, const Unit& u, int qi) {
    const int last = min((qi / p.head_tiles + 1) * p.tile_tokens, u.s.asked) - 1;
    const int seen = min(keys_seen(p, u.s, last, u.s.len, u.s.len) - u.k0, u.keys);
    return seen > 0 ? (seen + kTile - 1) / kTile : 0;
}

// The units of a CTA, the same for all its warps.
struct Units {
    int at;
    __device__ __forceinline__ Units() : at(blockIdx.x) {}
    __device__ __forceinline__ bool next(const MassParams& p, Unit& u) {
        for (; at < p.units; at += gridDim.x) {
            int x = at;
            u.id = at;
            u.h = x % p.kv_heads, x /= p.kv_heads;
            const int b = x % p.rows;
            x /= p.rows;
            const int c = x % p.chunks, split = x / p.chunks;
            u.s = sequence(p, b);
            u.k0 = c * p.chunk * kTile;
            u.keys = min(u.s.len - u.k0, p.chunk * kTile);
            if (u.keys <= 0) continue;
            u.tiles = (u.keys + kTile - 1) / kTile;
            const int all = row_tiles(p, u.s);
            u.q0 = split * p.split_tiles;
            u.q1 = min(u.q0 + p.split_tiles, all);
            // nothing to add: the join does not ask for the part, or the old weight stays
            if (p.splits > 1 ? u.q1 <= u.q0 || steps_of(p, u, u.q1 - 1) == 0 : u.s.n == 0 && p.decay == 1.f) continue;
            at += gridDim.x;
            return true;
        }
        return false;
    }
};

// Where a key's weight is kept; null where its page does not exist.
__device__ __forceinline__ float* mass_at(const MassParams& p, const Unit& u, int key) {
    int page, slot;
    locate(p, p.indices + u.s.page0, key, page, slot);
    return page < 0 ? nullptr : p.mass + page * p.m_page + slot * p.m_slot + u.h * p.m_head;
}
// Whether what a key has gathered is kept: not that of the call's own tokens, whose slots hold the
// weights of whoever had them before, and not where decay is 0.
__device__ __forceinline__ bool has_old(const MassParams& p, const Unit& u, int key) {
    return p.decay != 0.f && !(p.causal && key >= u.s.len - u.s.n);
}

__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        "\n\t}" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// DIM: head size rounded up to 64 elements; KSTEPS: 16 elements each.
template <typename T, int DIM, int KSTEPS>
__global__ void __launch_bounds__(kThreads, 1) mass_kernel(const __grid_constant__ MassParams p, const int box,
                                                           const __grid_constant__ CUtensorMap kmap,
                                                           const __grid_constant__ CUtensorMap qmap) {
    constexpr int kHalves = DIM / 64;
    constexpr int kBlock = kTile * DIM * 2;
    constexpr int kHalf = kTile * 128;
    extern __shared__ __align__(1024) unsigned char smem[];
    MassShared& sh = *reinterpret_cast<MassShared*>(smem + kTiles);
    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    const int q_half = p.tile_rows * 128, q_block = q_half * kHalves;
    const uint32_t sq = smem_addr(smem), ring = sq + p.q_bufs * q_block;
    const uint32_t b_full = smem_addr(sh.full), b_empty = smem_addr(sh.empty), b_qf = smem_addr(sh.q_full),
                   b_qe = smem_addr(sh.q_empty), b_if = smem_addr(sh.i_full), b_ie = smem_addr(sh.i_empty),
                   b_sf = smem_addr(sh.s_full), b_se = smem_addr(sh.s_empty);
    volatile int* fail = &sh.fail;

    if (warp == 9) {
        tmem_alloc(smem_addr(&sh.tmem), kCols);
        if (lane == 0) {
            for (int i = 0; i < kStagesMax; ++i) {
                mbar_init(&sh.full[i], 1);
                mbar_init(&sh.empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh.q_full[i], 1);
                mbar_init(&sh.q_empty[i], 1);
                mbar_init(&sh.i_full[i], 1);
                mbar_init(&sh.i_empty[i], 8);
                mbar_init(&sh.s_full[i], 1);
                mbar_init(&sh.s_empty[i], 4);
            }
            mbar_init(&sh.drained, 1);
            sh.fail = 0;
            fence_mbar_init();
        }
    }
    for (int i = tid; i < 2 * kChunkMax * kTile; i += kThreads) (&sh.acc[0][0])[i] = 0.f;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    Units units;
    Unit u;
    bool ok = true;

    if (warp == 9) {
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0 : 1;
        const uint32_t idesc = 1u << 4 | kType << 7 | kType << 10 | (kTile / 16) << 24 | (uint32_t)(p.tile_rows / 8) << 17;
        int f = 0, nq = 0;  // fills of the ring (steps) and row tiles so far
        while (ok && units.next(p, u)) {
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                const int steps = steps_of(p, u, qi);
                if (steps == 0) continue;
                const int qb = nq % p.q_bufs;
                ok = wait_warp(b_qf + qb * 8, nq / p.q_bufs & 1, fail);
                for (int j = 0; ok && j < steps; ++j, ++f) {
                    const int st = f % p.stages, w = f & 1;
                    ok = wait_warp(b_full + st * 8, f / p.stages & 1, fail) &&
                         (f < 2 || wait_warp(b_se + w * 8, (f / 2 - 1) & 1, fail));
                    if (!ok) break;
                    fence_after();
                    const uint32_t k = ring + st * kBlock, q = sq + qb * q_block;
#pragma unroll
                    for (int kk = 0; kk < KSTEPS; ++kk)
                        mma_ss(tmem + w * kMostRows, operand(k + (kk >> 2) * kHalf + (kk & 3) * 32, 16),
                               operand(q + (kk >> 2) * q_half + (kk & 3) * 32, 16), idesc, kk > 0);
                    commit(b_sf + w * 8);
                    commit(b_empty + st * 8);
                }
                if (ok) commit(b_qe + qb * 8);
                ++nq;
            }
        }
        if (!ok) {  // leave no product under way
            commit(smem_addr(&sh.drained));
            mbar_wait(&sh.drained, 0);
        }
    } else if (warp == 8) {
        // Lane l looks up the page of box l of a tile one tile ahead.  A box past the end is not
        // fetched; a page that does not exist is fetched from behind the last one, which reads as zeros.
        const int boxes = kTile / box;
        int f = 0;
        while (ok && units.next(p, u)) {
            const int64_t* list = p.indices + u.s.page0;
            const int end = u.k0 + u.keys;
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                const int steps = steps_of(p, u, qi);
                if (steps == 0) continue;
                int page, slot;
                auto find = [&](int at) {
                    page = -1, slot = 0;
                    if (at < end) {
                        locate(p, list, at, page, slot);
                        if (page < 0) page = p.pages;
                    }
                };
                if (lane < boxes) find(u.k0 + lane * box);
                for (int j = 0; j < steps; ++j, ++f) {
                    const int st = f % p.stages, kt = u.k0 + j * kTile;
                    const uint32_t dst = ring + st * kBlock, bar = b_full + st * 8;
                    if (f >= p.stages && !(ok = wait_warp(b_empty + st * 8, (f / p.stages - 1) & 1, fail))) break;
                    for (int b = 0; b < boxes; b += 32) {
                        if (b > 0) find(kt + (b + lane) * box);
                        const uint32_t held = __ballot_sync(kFull, lane < boxes - b && page >= 0);
                        if (lane == 0) {
                            const uint32_t bytes = __popc(held) * box * DIM * 2;
                            if (b + 32 >= boxes) mbar_arrive_expect_tx(&sh.full[st], bytes);
                            else mbar_expect_tx(&sh.full[st], bytes);
                        }
                        __syncwarp();
                        for (int i = 0; i < min(boxes - b, 32); ++i) {
                            const int pg = __shfl_sync(kFull, page, i), sl = __shfl_sync(kFull, slot, i);
                            if (!(held >> i & 1)) continue;
#pragma unroll
                            for (int half = 0; half < kHalves; ++half)
                                load_box(dst + half * kHalf + (b + i) * box * 128, &kmap, half * 64, sl, u.h, pg, bar);
                        }
                    }
                    if (lane < boxes) find(kt + kTile + lane * box);
                }
            }
        }
        __syncwarp();
        if (*fail)  // leave no copy under way
            for (int i = max(0, f - p.stages); i < f + p.stages; ++i)
                mbar_wait_brief(&sh.full[i % p.stages], i / p.stages & 1);
    } else if (warp == 10) {
        int nq = 0;
        while (ok && units.next(p, u)) {
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                if (steps_of(p, u, qi) == 0) continue;
                const int qb = nq % p.q_bufs, ib = nq & 1;
                const int t0 = qi / p.head_tiles * p.tile_tokens, h0 = qi % p.head_tiles * p.tile_heads;
                ok = nq < p.q_bufs || wait_warp(b_qe + qb * 8, (nq / p.q_bufs - 1) & 1, fail);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&sh.q_full[qb], p.tile_tokens * p.tile_heads * DIM * 2);
                __syncwarp();
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
                    load_box3(sq + qb * q_block + half * q_half, &qmap, half * 64, u.h * p.group + h0, u.s.first + t0, b_qf + qb * 8);
                ok = nq < 2 || wait_warp(b_ie + ib * 8, (nq / 2 - 1) & 1, fail);
                if (!ok) break;
                const int rows = min(p.tile_tokens, u.s.asked - t0) * p.tile_heads;
                int fewest = INT_MAX;
                for (int r = lane; r < ((rows + 31) & ~31); r += 32) {
                    const int i = t0 + r / p.tile_heads, x = h0 + r % p.tile_heads;
                    int seen = 0;
                    float l = 0.f;
                    if (r < rows && x < p.group) {
                        l = __ldg(p.row_lse + (int64_t)(u.s.first + i) * p.q_heads + u.h * p.group + x) * 1.4426950408889634f;
                        if (l != -INFINITY) seen = keys_seen(p, u.s, i, u.s.len, u.s.len);
                    }
                    sh.lse2[ib][r] = l;
                    sh.seen[ib][r] = seen;
                    if (r < rows) fewest = min(fewest, seen);
                }
                fewest = __reduce_min_sync(kFull, fewest);
                if (lane == 0) {
                    sh.fewest[ib] = fewest;
                    sh.rows[ib] = rows;
                }
                __syncwarp();
                if (lane == 0) arrive(b_if + ib * 8);
                ++nq;
            }
        }
        __syncwarp();
        if (*fail)
            for (int i = max(0, nq - 2); i <= nq; ++i) mbar_wait_brief(&sh.q_full[i % p.q_bufs], i / p.q_bufs & 1);
    } else if (warp < 8) {
        const int my = warp >> 2, key_of = tid & (kTile - 1);
        const uint32_t ts = tmem + my * kMostRows + ((uint32_t)(warp & 3) << 21);
        int f = 0, nq = 0;
        while (units.next(p, u)) {
            const bool direct = p.splits == 1 && u.q1 - u.q0 <= 1;
            auto add = [&](int key, float* at, float old, float sum) {
                if (at) *at = has_old(p, u, key) ? fmaf(old, p.decay, sum) : sum;
            };
            int done = 0;  // tiles of a direct unit that are written by their steps
            for (int qi = u.q0; ok && qi < u.q1; ++qi) {
                const int steps = steps_of(p, u, qi);
                if (steps == 0) continue;
                const int ib = nq & 1;
                ok = wait_warp(b_if + ib * 8, nq / 2 & 1, fail);
                const int rows = sh.rows[ib], fewest = sh.fewest[ib];
                for (int j = 0; ok && j < steps; ++j, ++f) {
                    if ((f & 1) != my) continue;
                    const int at = j * kTile + key_of, key = u.k0 + at;
                    float* to = nullptr;
                    float old = 0.f;
                    if (direct && at < u.keys) {
                        to = mass_at(p, u, key);
                        if (to && has_old(p, u, key)) old = *to;
                    }
                    ok = wait_warp(b_sf + my * 8, f / 2 & 1, fail);
                    fence_after();
                    const bool all = u.k0 + min((j + 1) * kTile, u.keys) <= fewest;  // every row sees every key
                    float sum = 0.f;
                    if (ok) {
#pragma unroll 1
                        for (int c = 0; c < rows; c += 32) {
                            uint32_t s[32];
                            tmem_ld32(ts + c, s);
                            wait_ld();
                            const float4* l4 = reinterpret_cast<const float4*>(&sh.lse2[ib][c]);
                            if (all && c + 32 <= rows) {
                                uint64_t part[2] = {0, 0};
                                const uint64_t sc = pair(p.scale_log2, p.scale_log2);
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    const float4 l = l4[e / 4];
                                    const float2 x = both(fma2(pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sc, pair(-l.x, -l.y)));
                                    const float2 y = both(fma2(pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), sc, pair(-l.z, -l.w)));
                                    part[0] = add2(part[0], pair(exp2_fast(x.x), exp2_fast(x.y)));
                                    part[1] = add2(part[1], pair(exp2_fast(y.x), exp2_fast(y.y)));
                                }
                                const float2 v = both(add2(part[0], part[1]));
                                sum += v.x + v.y;
                            } else {
                                const int4* n4 = reinterpret_cast<const int4*>(&sh.seen[ib][c]);
                                float part = 0.f;
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    const float4 l = l4[e / 4];
                                    const int4 n = n4[e / 4];
                                    part += key < n.x ? exp2_fast(fmaf(__uint_as_float(s[e]), p.scale_log2, -l.x)) : 0.f;
                                    part += key < n.y ? exp2_fast(fmaf(__uint_as_float(s[e + 1]), p.scale_log2, -l.y)) : 0.f;
                                    part += key < n.z ? exp2_fast(fmaf(__uint_as_float(s[e + 2]), p.scale_log2, -l.z)) : 0.f;
                                    part += key < n.w ? exp2_fast(fmaf(__uint_as_float(s[e + 3]), p.scale_log2, -l.w)) : 0.f;
                                }
                                sum += part;
                            }
                        }
                    } else {
                        sum = NAN;  // loud: a wait that ran out leaves no number
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(b_se + my * 8);
                    if (direct) add(key, to, old, sum);
                    else sh.acc[my][at] += sum;
                }
                __syncwarp();
                if (lane == 0) arrive(b_ie + ib * 8);
                ++nq;
                done = steps;
            }
            if (direct) {  // keys that no row sees
                for (int at = done * kTile + tid; at < u.keys; at += 2 * kTile) {
                    float* to = mass_at(p, u, u.k0 + at);
                    add(u.k0 + at, to, to && has_old(p, u, u.k0 + at) ? *to : 0.f, ok ? 0.f : NAN);
                }
                continue;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int at = tid; at < u.keys; at += 2 * kTile) {
                float sum = sh.acc[0][at] + sh.acc[1][at];
                if (!ok) sum = NAN;
                if (p.splits > 1) {
                    p.part[(int64_t)u.id * (p.chunk * kTile) + at] = sum;
                } else {
                    float* to = mass_at(p, u, u.k0 + at);
                    add(u.k0 + at, to, to && has_old(p, u, u.k0 + at) ? *to : 0.f, sum);
                }
            }
            // (keys behind the end were summed too)
            for (int at = tid; at < u.tiles * kTile; at += 2 * kTile) sh.acc[0][at] = sh.acc[1][at] = 0.f;
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 9) {
        fence_after();
        tmem_free(tmem, kCols);
    }
}

// mass of the keys of a (chunk, sequence, key head) from the parts of its row tiles, in their order.
__global__ void __launch_bounds__(256) mass_join_kernel(const __grid_constant__ MassParams p) {
    pdl_wait();
    Unit u;
    int x = blockIdx.x;
    u.h = x % p.kv_heads, x /= p.kv_heads;
    const int b = x % p.rows, c = x / p.rows;
    u.s = sequence(p, b);
    u.k0 = c * p.chunk * kTile;
    u.keys = min(u.s.len - u.k0, p.chunk * kTile);
    if (u.keys <= 0 || (u.s.n == 0 && p.decay == 1.f)) return;
    const int all = row_tiles(p, u.s), per = p.chunks * p.rows * p.kv_heads;
    for (int at = threadIdx.x; at < u.keys; at += blockDim.x) {
        float* const to = mass_at(p, u, u.k0 + at);
        if (!to) continue;
        float sum = 0.f;
        for (int s = 0; s < p.splits; ++s) {
            const int end = min((s + 1) * p.split_tiles, all);
            if (s * p.split_tiles >= end) break;
            if (steps_of(p, u, end - 1) == 0) continue;
            sum += p.part[((int64_t)s * per + blockIdx.x) * (p.chunk * kTile) + at];
        }
        *to = has_old(p, u, u.k0 + at) ? fmaf(*to, p.decay, sum) : sum;
    }
}

// ------------------------------------------------------------------ host
int make_plan(const tg_attention_mass_args* a, MassParams* out, const char* op) {
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
    const int64_t max_q = a->q_indptr ? std::min(a->max_q_len, a->tokens) : 1;

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

    // Row tiles: as many tokens as 256 rows hold (128 for heads of 256, whose tiles take twice the room),
    // or where one token's heads are more than that, a part of its heads.
    const int dim = (c.dim + 63) / 64 * 64, most = dim > 128 ? kMostRows / 2 : kMostRows;
    p.tile_heads = std::min(p.group, most);
    p.head_tiles = (p.group + p.tile_heads - 1) / p.tile_heads;
    p.tile_tokens = (int)std::max<int64_t>(1, std::min<int64_t>(max_q, most / p.tile_heads));
    p.tile_rows = (p.tile_tokens * p.tile_heads + 15) / 16 * 16;
    const int64_t q_tiles = std::max<int64_t>(1, ceil_div(max_q, p.tile_tokens)) * p.head_tiles, k_tiles = std::max<int64_t>(1, ceil_div(max_seq, kTile));
    // Chunks of keys: one row tile is loaded for each, so as long as leaves eight units a CTA; several row
    // tiles go over a chunk one after the other, its sums in shared memory.
    const int64_t pairs = std::max<int64_t>(1, t.rows * c.heads);
    p.chunk = (int)std::min<int64_t>(kChunkMax, q_tiles > 1 ? kChunkMax : std::max<int64_t>(1, pairs * k_tiles / (kSMs * 8)));
    p.chunks = (int)ceil_div(k_tiles, p.chunk);
    // Where that makes few units the row tiles are shared out too, at least two to a part.
    p.splits = (int)std::max<int64_t>(1, std::min(ceil_div(kSMs * 8, pairs * p.chunks), q_tiles / 2));
    p.split_tiles = (int)ceil_div(q_tiles, p.splits);
    p.splits = (int)std::max<int64_t>(1, ceil_div(q_tiles, p.split_tiles));
    if (pairs * p.chunks * p.splits > INT32_MAX - kSMs) return set_error(TG_EUNSUPPORTED, "%s: too many sequences for one launch", op);
    p.units = (int)(t.rows * c.heads * p.chunks * p.splits);
    const int q_block = p.tile_rows * dim * 2, k_block = kTile * dim * 2;
    p.q_bufs = 2 * q_block + 4 * k_block <= kTiles ? 2 : 1;
    p.stages = std::min(kStagesMax, (kTiles - p.q_bufs * q_block) / k_block);
    return TG_OK;
}

size_t mass_bytes(const MassParams& p) {
    return p.splits > 1 ? (size_t)p.units * p.chunk * kTile * sizeof(float) : 0;
}
// Of any smaller call: parts are made only until there are eight units an SM, rounded up by less than
// that.
size_t mass_enough(const MassParams& p) {
    const int64_t tiles = ceil_div(p.max_q, std::max(1, p.tile_tokens)) * p.head_tiles;
    return tiles < 2 && p.head_tiles < 2 ? 0 : (size_t)(2 * kSMs * 8) * kChunkMax * kTile * sizeof(float);
}

template <typename T, int DIM, int KSTEPS>
int mass_run(const MassParams& p, const CUtensorMap& kmap, const CUtensorMap& qmap, cudaStream_t st) {
    auto kernel = mass_kernel<T, DIM, KSTEPS>;
    static SmemOnce once;
    int rc = once.raise(reinterpret_cast<const void*>(kernel), kSmem);
    if (rc != TG_OK) return rc;
    const int grid = std::min(p.units, kSMs);
    kernel<<<(unsigned)grid, kThreads, kSmem, st>>>(p, std::gcd(p.page_size, kTile), kmap, qmap);
    rc = check_launch("mass_kernel");
    if (rc != TG_OK || p.splits == 1) return rc;
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
    if (ws_bytes < need || (need && !ws)) return set_error(TG_EINVAL, "%s: workspace of %zu bytes needed (got %zu)", op, need, ws_bytes);
    if (reinterpret_cast<uintptr_t>(ws) % 16) return set_error(TG_EINVAL, "%s: the workspace must be 16-byte aligned", op);
    p.part = static_cast<float*>(ws);
    constexpr bool kIsHalf = std::is_same<T, __half>::value;
    CUtensorMap kmap, vmap, qmap;
    rc = cache_maps(p, kIsHalf, c.dim, std::gcd(p.page_size, kTile), &kmap, &vmap);
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
    return tg::make_plan(a, &p, "tg_attention_mass") == TG_OK ? tg::mass_enough(p) : 0;
}

int tg_attention_mass_f16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::attention_mass<__half>(a, workspace, workspace_bytes, stream, "tg_attention_mass_f16");
}

int tg_attention_mass_bf16(const tg_attention_mass_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::attention_mass<__nv_bfloat16>(a, workspace, workspace_bytes, stream, "tg_attention_mass_bf16");
}

}  // extern "C"
