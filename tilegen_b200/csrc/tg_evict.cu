// Eviction from a paged cache by the weight that keys have gathered (tg_kv_evict_*).
//
// A sequence longer than the budget is cut to it: its first places, its recent (last) ones and, for
// each key head by itself, the heaviest of those between stay; ties go to the lowest place.  With
// `heavy` = budget - first - recent the new places are
//   [0, first)                     what they were,
//   [first, first + heavy)         the chosen keys: those that lie here already stay, the others fill
//                                  the holes, both in the order of their places,
//   [budget - recent, budget)      the recent ones, moved down, in their order.
// So about half of what a compaction in order would move is moved, or one key and the recent ones for
// a sequence one over its budget; attention does not depend on the order of keys that carry their
// positions.
//
// * select_kernel: a cluster of CTAs for each (sequence, key head).  Weights as ordered 32-bit
//   integers lie in shared memory; four rounds of 11, 8, 8 and 5 bits find the value of the heavy-th
//   largest (histograms of all CTAs, added over the cluster), the last two over the keys that begin
//   like it, which each warp lists in the second (over all keys again in a CTA where a warp's list
//   overflows); then ranks in the order of the places give the holes and the keys that fill them.
//   Bound: latency.  512 (sequence, head) pairs of 1000 keys 11 us, two sequences of 120000 (clusters of
//   eight CTAs, 15000 keys each) 50 us: reading 8, histograms 12, their sums over the cluster 12, ranks
//   and lists 15.
// * move_kernel: holes are filled from places behind the budget by all CTAs side by side: such places are
//   not written, so nothing waits.  Sources before the budget lie where recent keys go: these fills
//   and the recent keys are one list, sorted so that a place is read before it is written, that the
//   CTAs of one cluster go through together, reading a batch before it writes it.  Bound: HBM with
//   rows of 256 bytes from pages in random order: 224 MB in 42 us, 5.3 TB/s.
#include <cooperative_groups.h>

#include <algorithm>

#include "tg_paged.cuh"

namespace tg {
namespace {

namespace cg = cooperative_groups;

constexpr int kBins = 2048;
constexpr int kSelKeys = 40960;  // most weights of a CTA in shared memory; further ones are read again
constexpr int kMoveThreads = 256;
constexpr int kListed = 2048; // keys of one beginning that are listed
constexpr int kMostCtas = 8;  // of a cluster

struct EvictParams {
    tg_csr pages;
    int64_t page_size;
    int page_shift;  // log2(page_size), -1 where it is no power of two
    const int64_t* seq_len;
    int64_t *seq_len_out, n_pages;
    int max_seq, budget, first, recent, heads, rows;
    const float* mass;
    float* mass_out;
    int64_t m_page, m_slot, m_head, mo_page, mo_slot, mo_head;
    int32_t* kept;  // [sequence][head][kept_width] or null
    int kept_width;
    char *k, *v;  // strides in bytes
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int row_bytes, moved;  // moved: mass_out is not mass
    // workspace: of each (sequence, head) its counts, holes and the places of what fills them
    int4* counts;  // fills, those of them from places before the new length, new length, places gone
    int* holes;
    int* fills;
    int width;  // places of each
    int parts;  // clusters of the move for each (sequence, head)
};

// A sequence as it is cut: its parts of a length.
struct Cut {
    int len, size, gone, first, recent, heavy;
};
__device__ __forceinline__ Cut cut_of(const EvictParams& p, int64_t b, int64_t& page0) {
    int64_t npages;
    pages_of(p.pages.indptr, p.pages.nnz, b, page0, npages);
    Cut c;
    const int64_t len = min(min(p.seq_len[b], npages * p.page_size), (int64_t)p.max_seq);
    c.len = (int)max(len, (int64_t)0);
    c.size = min(c.len, p.budget);
    c.gone = c.len - c.size;
    c.recent = min(p.recent, c.size);
    c.first = min(p.first, c.size - c.recent);
    c.heavy = c.size - c.recent - c.first;
    return c;
}

struct Place {
    int page, slot;  // page -1: not in the cache
};
__device__ __forceinline__ int page_index(const EvictParams& p, int at) {
    return p.page_shift >= 0 ? at >> p.page_shift : at / (int)p.page_size;
}
__device__ __forceinline__ Place place_of(const EvictParams& p, int64_t page0, int at) {
    const int j = page_index(p, at);
    const int64_t id = __ldg(p.pages.indices + page0 + j);
    return {id >= 0 && id < p.n_pages ? (int)id : -1, at - j * (int)p.page_size};
}
__device__ __forceinline__ float mass_of(const EvictParams& p, int64_t page0, int at, int h) {
    const Place x = place_of(p, page0, at);
    return x.page < 0 ? 0.f : p.mass[x.page * p.m_page + x.slot * p.m_slot + h * p.m_head];
}
__device__ __forceinline__ void put_mass(const EvictParams& p, int64_t page0, int at, int h, float v) {
    const Place x = place_of(p, page0, at);
    if (x.page >= 0) p.mass_out[x.page * p.mo_page + x.slot * p.mo_slot + h * p.mo_head] = v;
}
// Weights in their order as integers; the two zeros are one, NaN is above all.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums over the warps before mine, and over all, of three numbers (the same in all lanes of a warp).
struct Before {
    int3 mine, all;
};
template <int WARPS>
__device__ __forceinline__ Before warps_before(int3 v, int3* s) {  // s: [WARPS]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) s[warp] = v;
    __syncthreads();
    const int3 x = lane < WARPS ? s[lane] : make_int3(0, 0, 0);
    const bool before = lane < warp;
    Before r;
    r.mine = make_int3(__reduce_add_sync(kFull, before ? x.x : 0), __reduce_add_sync(kFull, before ? x.y : 0),
                       __reduce_add_sync(kFull, before ? x.z : 0));
    r.all = make_int3(__reduce_add_sync(kFull, x.x), __reduce_add_sync(kFull, x.y), __reduce_add_sync(kFull, x.z));
    return r;
}
// The same over the CTAs of a cluster (32 at most), of what they write into *s.
__device__ __forceinline__ Before ctas_before(cg::cluster_group& cl, int3 v, int3* s) {
    if (cl.num_blocks() == 1) return {make_int3(0, 0, 0), v};
    cl.sync();  // the last values have been read
    if (threadIdx.x == 0) *s = v;
    cl.sync();
    const unsigned lane = threadIdx.x & 31;
    const int3 x = lane < cl.num_blocks() ? *cl.map_shared_rank(s, lane) : make_int3(0, 0, 0);
    const bool before = lane < cl.block_rank();
    Before r;
    r.mine = make_int3(__reduce_add_sync(kFull, before ? x.x : 0), __reduce_add_sync(kFull, before ? x.y : 0),
                       __reduce_add_sync(kFull, before ? x.z : 0));
    r.all = make_int3(__reduce_add_sync(kFull, x.x), __reduce_add_sync(kFull, x.y), __reduce_add_sync(kFull, x.z));
    return r;
}

// THREADS: 256 where a CTA has up to 4096 candidates, whose time goes into scans of all warps, else 512 (with
// 1024, of which an SM holds one CTA, sixteen clusters of eight did not fit at once: 80 us for two long
// sequences).
template <int THREADS>
__global__ void __launch_bounds__(THREADS) select_kernel(const __grid_constant__ EvictParams p, const int held) {
    constexpr int kWarps = THREADS / 32, kLoads = 8;                  // weights of a thread under way
    constexpr int kList = kListed / kWarps;  // places of a warp's list
    extern __shared__ float s_mass[];  // [held]
    __shared__ uint32_t s_hist[kBins], s_total[kBins];  // s_total: of the cluster
    __shared__ int3 s_warp[kWarps], s_cta;
    __shared__ int s_pick[3], s_over;
    __shared__ uint32_t s_list[kListed];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int ctas = cl.num_blocks(), rank = cl.block_rank();
    auto sync = [&] {
        if (ctas == 1) __syncthreads();
        else cl.sync();
    };
    pdl_trigger();
    const int unit = blockIdx.x / ctas, h = unit % p.heads, b = unit / p.heads;
    int64_t page0;
    const Cut c = cut_of(p, b, page0);
    const int new_end = c.first + c.heavy;  // of the new places of the chosen ones

    // what stays where it is, and the ends of the lists
    int32_t* const kept = p.kept ? p.kept + ((int64_t)b * p.heads + h) * p.kept_width : nullptr;
    auto stays = [&](int at, float m) {
        if (p.moved) put_mass(p, page0, at, h, m);
        if (kept) kept[at] = at;
    };
    const int step = ctas * THREADS, me = rank * THREADS + tid;
    if (kept)
        for (int at = c.size + me; at < p.kept_width; at += step) kept[at] = -1;
    auto first_stay = [&] {
        if (p.moved || kept)
            for (int at = me; at < (c.gone ? c.first : c.size); at += step) stays(at, p.moved ? mass_of(p, page0, at, h) : 0.f);
    };
    if (c.gone == 0 || c.heavy == 0) {  // the same for the whole cluster
        first_stay();
        if (me == 0) p.counts[unit] = make_int4(0, 0, c.size, c.gone);
        return;
    }

    // my share of the candidates, a multiple of 32 for each warp
    const int all = c.len - c.recent - c.first;
    const int per_warp = ((all + ctas * kWarps - 1) / (ctas * kWarps) + 31) & ~31, per = per_warp * kWarps;
    const int lo = min(rank * per, all), n = min(lo + per, all) - lo;  // candidates lo .. lo + n, from place c.first
    const int base = c.first + lo;
    // several pages, then several weights under way (of a place that is none, some)
    for (int i0 = tid; i0 < min(n, held); i0 += kLoads * THREADS) {
        int64_t id[kLoads];
        float m[kLoads];
        bool there[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) id[k] = __ldg(p.pages.indices + page0 + page_index(p, base + min(i0 + k * THREADS, n - 1)));
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int at = base + min(i0 + k * THREADS, n - 1), slot = at - page_index(p, at) * (int)p.page_size;
            there[k] = id[k] >= 0 && id[k] < p.n_pages;
            m[k] = __ldg(p.mass + (there[k] ? id[k] : 0) * p.m_page + slot * p.m_slot + h * p.m_head);
        }
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (i0 + k * THREADS < min(n, held)) s_mass[i0 + k * THREADS] = there[k] ? m[k] : 0.f;
    }
    auto mass = [&](int i) { return i < held ? s_mass[i] : mass_of(p, page0, base + i, h); };

    // The value of the heavy-th largest, from its high bits on: 11 of them, then 8, 8 and 5 of the keys that
    // begin alike, which the second round lists (where they are not too many).
    uint32_t prefix = 0;
    int need = c.heavy, alike = 0;  // how many of those that begin with the prefix are chosen, and are there
    // the bin of the need-th key from above, over all CTAs; EACH bins a thread
    auto pick = [&](int bins, int shift, auto each_) {
        constexpr int EACH = decltype(each_)::value;
        const uint32_t* hist = s_hist;
        if (ctas > 1) {
            // each CTA adds a share of the bins of all, then everyone takes all shares: in steps of whole lines,
            // as other CTAs' memory is read slowly otherwise
            const int part = bins / ctas;
            for (int i = tid; i < part; i += THREADS) {
                uint32_t sum = 0;
#pragma unroll
                for (int r = 0; r < kMostCtas; ++r)
                    if (r < ctas) sum += cl.map_shared_rank(s_hist, r)[rank * part + i];
                s_total[rank * part + i] = sum;
            }
            cl.sync();
#pragma unroll 4
            for (int i = tid; i < bins; i += THREADS)
                if (i / part != rank) s_total[i] = cl.map_shared_rank(s_total, i / part)[i];
            __syncthreads();
            hist = s_total;
        }
        const int bin0 = bins - EACH - tid * EACH;
        uint32_t v[EACH] = {};
        if (bin0 >= 0)
#pragma unroll
            for (int i = 0; i < EACH; ++i) v[i] = hist[bin0 + i];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) mine += (int)v[i];
        int scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(kFull, scan, o);
            if (lane >= o) scan += x;
        }
        if (lane == 31) s_warp[warp].x = scan;
        __syncthreads();
        const int below = __reduce_add_sync(kFull, lane < warp ? s_warp[lane].x : 0);
        int higher = below + scan - mine;  // keys in the bins above mine
        if (higher < need && higher + mine >= need) {
#pragma unroll
            for (int i = EACH - 1; i >= 0; --i) {
                if (higher < need && higher + (int)v[i] >= need) s_pick[0] = bin0 + i, s_pick[1] = need - higher, s_pick[2] = v[i];
                higher += v[i];
            }
        }
        sync();  // the histograms have been read
        prefix |= (uint32_t)s_pick[0] << shift;
        need = s_pick[1], alike = s_pick[2];
    };
    int listed = 0;  // by my warp
    uint32_t* const list = s_list + warp * kList;
#pragma unroll 1
    for (int round = 0; round < 4; ++round) {
        const int bits = round == 0 ? 11 : round < 3 ? 8 : 5, shift = round == 0 ? 21 : round == 1 ? 13 : round == 2 ? 5 : 0;
        const uint32_t above = round == 0 ? 0u : ~0u << (shift + bits), mask = (1u << bits) - 1;
        for (int i = tid; i < 1 << bits; i += THREADS) s_hist[i] = 0;
        if (tid == 0 && round == 0) s_over = 0;
        __syncthreads();
        if (round > 1 && !s_over) {
            for (int i = lane; i < listed; i += 32)
                if ((list[i] & above) == prefix) atomicAdd(&s_hist[list[i] >> shift & mask], 1u);
        } else {
#pragma unroll 4
            for (int i0 = 0; i0 < n; i0 += THREADS) {
                const uint32_t k = i0 + tid < n ? ordered(mass(i0 + tid)) : 0u;
                const bool same = i0 + tid < n && (k & above) == prefix;
                if (same) atomicAdd(&s_hist[k >> shift & mask], 1u);
                if (round == 1) {
                    const uint32_t all_same = __ballot_sync(kFull, same);
                    const int at = listed + __popc(all_same & ((1u << lane) - 1));
                    if (same && at < kList) list[at] = k;
                    listed += __popc(all_same);
                }
            }
            if (round == 1 && listed > kList) s_over = 1;
            __syncwarp();
        }
        sync();
        if (round == 0) pick(1 << bits, shift, std::integral_constant<int, kBins / THREADS>());
        else pick(1 << bits, shift, std::integral_constant<int, 1>());
    }

    // A warp's places are consecutive.  Equal ones are chosen from the lowest place on: how many lie
    // before the warp's?
    const int w0 = min(warp * per_warp, n), w1 = min(w0 + per_warp, n);
    int equal0 = 0;
    if (need < alike) {  // the same for the whole cluster
        int equal = 0;
        for (int i = w0; i < w1; i += 32) equal += __popc(__ballot_sync(kFull, i + lane < w1 && ordered(mass(i + lane)) == prefix));
        const Before wb = warps_before<kWarps>(make_int3(equal, 0, 0), s_warp), cb = ctas_before(cl, wb.all, &s_cta);
        equal0 = cb.mine.x + wb.mine.x;
    }
    // Walks the warp's places, kStep times 32 at a time: what(places, chosen, weights).
    const bool ties = need < alike;
    constexpr int kStep = 4;
    auto walk = [&](auto what) {
        int eq = equal0;
        for (int i = w0; i < w1; i += 32 * kStep) {
            float m[kStep];
            bool chosen[kStep];
#pragma unroll
            for (int k = 0; k < kStep; ++k) m[k] = i + k * 32 + lane < w1 ? mass(i + k * 32 + lane) : 0.f;
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
                const bool in = i + k * 32 + lane < w1;
                const uint32_t x = ordered(m[k]);
                chosen[k] = in && x >= prefix;
                if (ties) {
                    const uint32_t same = __ballot_sync(kFull, in && x == prefix);
                    chosen[k] = in && (x > prefix || (x == prefix && eq + __popc(same & ((1u << lane) - 1)) < need));
                    eq += __popc(same);
                }
            }
            what(base + i + lane, chosen, m);
        }
    };
    const int place_end = base + w1;
    int3 sums = make_int3(0, 0, 0);  // holes, those that fill them, those of them from places before the new length
    walk([&](int at, const bool (&chosen)[kStep], const float (&)[kStep]) {
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            const bool front = at + k * 32 < new_end;
            sums.x += front && !chosen[k] && at + k * 32 < place_end;
            sums.y += chosen[k] && !front;
            sums.z += chosen[k] && !front && at + k * 32 < c.size;
        }
    });
    sums = make_int3(__reduce_add_sync(kFull, sums.x), __reduce_add_sync(kFull, sums.y), __reduce_add_sync(kFull, sums.z));
    const Before wb = warps_before<kWarps>(sums, s_warp), cb = ctas_before(cl, wb.all, &s_cta);
    int hole_at = cb.mine.x + wb.mine.x, move_at = cb.mine.y + wb.mine.y;
    if (me == 0) p.counts[unit] = make_int4(cb.all.y, cb.all.z, c.size, c.gone);
    int* const hole_list = p.holes + (int64_t)unit * p.width;
    int* const fill_list = p.fills + (int64_t)unit * p.width;
    walk([&](int at, const bool (&chosen)[kStep], const float (&m)[kStep]) {
        const uint32_t below = (1u << lane) - 1;
        // most warps are on one side of the new places' end
        if (at - lane + 32 * kStep > new_end) {
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
                const bool moves = chosen[k] && at + k * 32 >= new_end;
                const uint32_t move = __ballot_sync(kFull, moves);
                if (moves) fill_list[move_at + __popc(move & below)] = at + k * 32;
                move_at += __popc(move);
            }
        }
        if (at - lane >= new_end) return;
        bool stay[kStep];
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            const bool front = at + k * 32 < new_end, is_hole = front && !chosen[k] && at + k * 32 < place_end;
            const uint32_t hole = __ballot_sync(kFull, is_hole);
            if (is_hole) hole_list[hole_at + __popc(hole & below)] = at + k * 32;
            hole_at += __popc(hole);
            stay[k] = chosen[k] && front;
        }
        if (!p.moved && !kept) return;
        Place x[kStep];
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            x[k].page = -1;
            if (p.moved && stay[k]) x[k] = place_of(p, page0, at + k * 32);
        }
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            if (x[k].page >= 0) p.mass_out[x[k].page * p.mo_page + x[k].slot * p.mo_slot + h * p.mo_head] = m[k];
            if (kept && stay[k]) kept[at + k * 32] = at + k * 32;
        }
    });
    first_stay();
    if (ctas > 1) cl.sync();  // no CTA leaves while its counts are read
}

// Words of U bytes.
template <int U>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<2> { using type = uint16_t; };

template <int U>
__global__ void __launch_bounds__(kMoveThreads, 4) move_kernel(const __grid_constant__ EvictParams p) {
    using W = typename Word<U>::type;
    constexpr int kAhead = 8;  // words of a thread under way
    // of each staged move: bytes from the head's first element to its old and new rows of k and of v, -1:
    // no such page
    __shared__ int64_t s_k[2][kMoveThreads], s_v[2][kMoveThreads];
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = cl.num_blocks(), rank = cl.block_rank();
    const int cluster = blockIdx.x / ctas, part = cluster % p.parts, unit = cluster / p.parts;
    const int h = unit % p.heads, b = unit / p.heads, tid = threadIdx.x;
    const int words = p.row_bytes / U, lanes = min(2 * words, kMoveThreads), groups = kMoveThreads / lanes, group = tid / lanes,
              lane = tid - group * lanes;
    const int ahead = min(kAhead, kMoveThreads / groups), batch = groups * ahead;  // rows of a CTA under way
    const int staged = kMoveThreads / batch * batch;
    pdl_wait();
    const int4 n = p.counts[unit];
    const int fills = n.x, early = n.y, size = n.z, gone = n.w;
    if (part == 0 && h == 0 && rank == 0 && tid == 0) p.seq_len_out[b] = size;
    if (gone == 0) return;
    int64_t page0, npages;
    pages_of(p.pages.indptr, p.pages.nnz, b, page0, npages);
    const int recent = min(p.recent, size);
    const int* const hole_list = p.holes + (int64_t)unit * p.width;
    const int* const fill_list = p.fills + (int64_t)unit * p.width;
    int32_t* const kept = p.kept ? p.kept + ((int64_t)b * p.heads + h) * p.kept_width : nullptr;
    char *const k0 = p.k + h * p.k_head, *const v0 = p.v + h * p.v_head;

    // The list: the early fills, the recent keys, then the other fills.  Part 0 goes through the first two
    // in order, a batch of the cluster read before it is written, and through all where it is the only
    // part; the others share the rest.
    const bool in_order = part == 0;
    const int all = recent + fills, ordered_end = p.parts == 1 ? all : early + recent;
    const int rest = all - ordered_end, shares = max(1, (p.parts - 1) * ctas), share = (part - 1) * ctas + rank;
    const int begin = in_order ? 0 : ordered_end + (int)((int64_t)rest * share / shares);
    const int end = in_order ? ordered_end : ordered_end + (int)((int64_t)rest * (share + 1) / shares);
    const int spread = in_order ? ctas : 1;  // CTAs that share a batch
    for (int at = begin; at < end; at += staged * spread) {
        // move `tid` of mine: its places, weight and number
        const int s = tid / batch, i = at + (s * spread + (in_order ? rank : 0)) * batch + tid - s * batch;
        const bool mine = tid < staged && i < end;
        int to = 0, from = 0;
        float m = 0.f;
        __syncthreads();  // the places before have been used
        if (mine) {
            if (i < early || i >= early + recent) {
                const int f = i < early ? i : i - recent;
                to = hole_list[f], from = fill_list[f];
            } else {
                to = size - recent + i - early, from = to + gone;
            }
            const Place x = place_of(p, page0, from), y = place_of(p, page0, to);
            s_k[0][tid] = x.page < 0 ? -1 : x.page * p.k_page + x.slot * p.k_slot;
            s_v[0][tid] = x.page < 0 ? -1 : x.page * p.v_page + x.slot * p.v_slot;
            s_k[1][tid] = y.page < 0 ? -1 : y.page * p.k_page + y.slot * p.k_slot;
            s_v[1][tid] = y.page < 0 ? -1 : y.page * p.v_page + y.slot * p.v_slot;
            m = x.page < 0 ? 0.f : p.mass[x.page * p.m_page + x.slot * p.m_slot + h * p.m_head];
        }
        __syncthreads();
        bool first = true;
        for (int w0 = 0; w0 < 2 * words; w0 += lanes) {
            const int word = w0 + lane;
            const bool is_v = word >= words, has = group < groups && word < 2 * words;
            const int64_t* const where = is_v ? s_v[0] : s_k[0];
            char* const rows = (is_v ? v0 : k0) + (int64_t)(is_v ? word - words : word) * U;
            for (int r0 = 0; r0 < staged; r0 += batch) {
                const int left = end - (at + (r0 / batch * spread + (in_order ? rank : 0)) * batch);  // of the list, from this batch on
                if (in_order ? end <= at + r0 * spread : left <= 0) break;                            // the same for the cluster
                W w[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int r = group + k * groups;
                    memset(&w[k], 0, sizeof(W));
                    if (k < ahead && has && r < left && where[r0 + r] >= 0) w[k] = *reinterpret_cast<const W*>(rows + where[r0 + r]);
                }
                if (in_order) {
                    if (ctas == 1) __syncthreads();
                    else cl.sync();
                }
                if (first && mine) {
                    put_mass(p, page0, to, h, m);
                    if (kept) kept[to] = from;
                }
                first = false;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int r = group + k * groups;
                    if (k < ahead && has && r < left && where[kMoveThreads + r0 + r] >= 0)
                        *reinterpret_cast<W*>(rows + where[kMoveThreads + r0 + r]) = w[k];
                }
            }
        }
    }
}

// ------------------------------------------------------------------ host
struct Plan {
    EvictParams p;
    int unit;           // bytes moved at once
    int select_ctas, select_threads, move_ctas;
    int held;
    size_t bytes, counts_bytes;
};

int make_plan(const tg_kv_evict_args* a, int elem, Plan* plan, const char* op) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_cache(a->cache, op);
    if (rc == TG_OK && !a->pages) rc = set_error(TG_EINVAL, "%s: null page table", op);
    if (rc != TG_OK) return rc;
    const tg_paged_kv& c = *a->cache;
    const tg_csr& t = *a->pages;
    if (t.rows < 0 || t.rows > INT32_MAX || t.nnz < 0)
        return set_error(TG_EINVAL, "%s: bad size (sequences=%lld pages=%lld)", op, (long long)t.rows, (long long)t.nnz);
    if (t.cols != c.pages)
        return set_error(TG_EINVAL, "%s: the page table has %lld columns and the cache %lld pages", op, (long long)t.cols,
                         (long long)c.pages);
    if (a->max_seq_len < 0 || a->budget < 0 || a->first < 0 || a->recent < 0)
        return set_error(TG_EINVAL, "%s: negative max_seq_len, budget, first or recent", op);
    if (a->flags & ~TG_FLAG_BOUNDS_CHECK) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if (c.dim > 1 << 24) return set_error(TG_EUNSUPPORTED, "%s: heads of more than 2^24 elements (got %d)", op, c.dim);
    if (a->kept && a->kept_width < 0) return set_error(TG_EINVAL, "%s: negative kept_width", op);
    const int64_t slots = c.pages == 0 ? 0 : t.nnz > INT32_MAX / c.page_size ? INT32_MAX / 2 : t.nnz * c.page_size;
    const int64_t max_seq = std::min({a->max_seq_len, slots, (int64_t)INT32_MAX / 2});
    EvictParams& p = plan->p;
    p = {};
    p.pages = t, p.page_size = c.page_size, p.n_pages = c.pages;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (c.page_size == (1ll << i)) p.page_shift = i;
    p.seq_len = a->seq_len, p.seq_len_out = a->seq_len_out;
    p.max_seq = (int)max_seq;
    p.budget = (int)std::min<int64_t>(a->budget, INT32_MAX / 2);
    p.first = (int)std::min<int64_t>(a->first, INT32_MAX / 2), p.recent = (int)std::min<int64_t>(a->recent, INT32_MAX / 2);
    p.heads = c.heads, p.rows = (int)t.rows;
    const int64_t units = t.rows * c.heads;
    p.mass = a->mass.data, p.mass_out = a->mass_out.data ? a->mass_out.data : a->mass.data;
    p.m_page = stride_of(c.pages, a->mass.page_stride), p.m_slot = stride_of(c.page_size, a->mass.slot_stride);
    p.m_head = stride_of(c.heads, a->mass.head_stride);
    const tg_paged_mass& mo = a->mass_out.data ? a->mass_out : a->mass;
    p.mo_page = stride_of(c.pages, mo.page_stride), p.mo_slot = stride_of(c.page_size, mo.slot_stride);
    p.mo_head = stride_of(c.heads, mo.head_stride);
    p.moved = p.mass_out != p.mass;
    p.kept = a->kept, p.kept_width = (int)std::min<int64_t>(a->kept_width, INT32_MAX / 2);
    p.k = static_cast<char*>(c.k), p.v = static_cast<char*>(c.v);
    p.k_page = stride_of(c.pages, c.k_page_stride) * elem, p.v_page = stride_of(c.pages, c.v_page_stride) * elem;
    p.k_slot = stride_of(c.page_size, c.k_slot_stride) * elem, p.v_slot = stride_of(c.page_size, c.v_slot_stride) * elem;
    p.k_head = stride_of(c.heads, c.k_head_stride) * elem, p.v_head = stride_of(c.heads, c.v_head_stride) * elem;
    p.row_bytes = c.dim * elem;
    const uint64_t all = reinterpret_cast<uint64_t>(p.k) | reinterpret_cast<uint64_t>(p.v) |
                         (uint64_t)(p.k_page | p.k_slot | p.k_head | p.v_page | p.v_slot | p.v_head | p.row_bytes);
    plan->unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
    // most places of a sequence that fill a hole: as many as it loses, and as the chosen ones are
    const int64_t gone = std::max<int64_t>(0, max_seq - p.budget);
    p.width = (int)std::min<int64_t>(gone, p.budget);
    // The selection: 8192 candidates a CTA, and more CTAs where few pairs leave SMs idle.
    const int64_t most = gone > 0 ? max_seq : 0;
    plan->select_ctas = 1;
    while (plan->select_ctas < kMostCtas && (most > 8192ll * plan->select_ctas ||
                                             (most > 2048ll * plan->select_ctas && units * plan->select_ctas * 2 <= kSMs)))
        plan->select_ctas *= 2;
    const int64_t each = ceil_div(most, plan->select_ctas);
    plan->select_threads = each > 4096 ? 512 : 256;
    plan->held = (int)std::min<int64_t>(kSelKeys, ceil_div(each, plan->select_threads) * plan->select_threads);
    // The move: the list in order by a cluster of up to eight CTAs, 64 rows each at once; the other
    // fills in parts of 64 rows and more, about eight CTAs an SM in all, or at the end of the list where
    // they are few.
    const int64_t in_order = std::min<int64_t>(p.recent, p.budget) * 2;
    plan->move_ctas = 1;
    while (plan->move_ctas < kMostCtas && in_order > 128ll * plan->move_ctas) plan->move_ctas *= 2;
    const int64_t want = std::min(ceil_div(p.width, 64 * plan->move_ctas),
                                  std::max<int64_t>(1, kSMs * 8 / std::max<int64_t>(1, units * plan->move_ctas)));
    p.parts = 1 + (p.width > 32 ? (int)std::max<int64_t>(1, want) : 0);
    if (units * std::max(p.parts * plan->move_ctas, plan->select_ctas) > INT32_MAX)
        return set_error(TG_EUNSUPPORTED, "%s: too many sequences for one launch", op);
    plan->counts_bytes = ((size_t)units * sizeof(int4) + 255) / 256 * 256;
    plan->bytes = plan->counts_bytes + (size_t)units * p.width * 2 * sizeof(int);
    return TG_OK;
}

template <typename... P, typename... A>
int launch_clusters(const char* what, void (*kernel)(P...), int64_t grid, int block, int cluster, size_t smem, bool pdl,
                    cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    const int rc = check_launch(what);
    return e != cudaSuccess ? check_cuda(e, what) : rc;
}

int evict(const tg_kv_evict_args* a, int elem, void* ws, size_t ws_bytes, tg_stream_t stream, const char* op) {
    Plan plan;
    int rc = make_plan(a, elem, &plan, op);
    if (rc != TG_OK) return rc;
    EvictParams& p = plan.p;
    if (p.rows == 0) return TG_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!a->seq_len || !a->seq_len_out || !a->pages->indptr) return set_error(TG_EINVAL, "%s: null indptr/seq_len/seq_len_out", op);
    if (a->pages->nnz > 0 && !a->pages->indices) return set_error(TG_EINVAL, "%s: null page indices", op);
    if (a->cache->pages > 0 && !p.mass) return set_error(TG_EINVAL, "%s: null mass", op);
    if (a->kept && p.kept_width < std::min<int64_t>(p.budget, p.max_seq))
        return set_error(TG_EINVAL, "%s: kept has %d places, not the %lld that may be kept", op, p.kept_width,
                         (long long)std::min<int64_t>(p.budget, p.max_seq));
    if (a->flags & TG_FLAG_BOUNDS_CHECK) {
        rc = paged_bounds_check(*a->pages, p.page_size, a->seq_len, a->max_seq_len, p.rows, nullptr, 1, nullptr, 0, false, op, st);
        if (rc != TG_OK) return rc;
    }
    if (ws_bytes < plan.bytes || (plan.bytes && !ws))
        return set_error(TG_ENOMEM, "%s: workspace of %zu bytes needed (got %zu)", op, plan.bytes, ws_bytes);
    if (reinterpret_cast<uintptr_t>(ws) % 16) return set_error(TG_EINVAL, "%s: the workspace must be 16-byte aligned", op);
    p.counts = static_cast<int4*>(ws);
    p.holes = reinterpret_cast<int*>(static_cast<char*>(ws) + plan.counts_bytes);
    p.fills = p.holes + (int64_t)p.rows * p.heads * p.width;
    const int64_t units = (int64_t)p.rows * p.heads;
    const size_t smem = (size_t)plan.held * sizeof(uint32_t);
    auto select = plan.select_threads == 256 ? select_kernel<256> : select_kernel<512>;
    static SmemOnce once[2];
    rc = once[plan.select_threads == 256].raise(reinterpret_cast<const void*>(select), kSelKeys * (int)sizeof(uint32_t));
    if (rc != TG_OK) return rc;
    rc = launch_clusters("select_kernel", select, units * plan.select_ctas, plan.select_threads, plan.select_ctas, smem, false, st, p,
                         plan.held);
    if (rc != TG_OK) return rc;
    auto kernel = plan.unit == 16 ? move_kernel<16> : plan.unit == 4 ? move_kernel<4> : move_kernel<2>;
    return launch_clusters("move_kernel", kernel, units * p.parts * plan.move_ctas, kMoveThreads, plan.move_ctas, 0, true, st, p);
}

}  // namespace
}  // namespace tg

extern "C" {

size_t tg_kv_evict_workspace_bytes(const tg_kv_evict_args* a) {
    tg::Plan plan;
    return tg::make_plan(a, 4, &plan, "tg_kv_evict") == TG_OK ? plan.bytes : 0;
}

int tg_kv_evict_f32(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::evict(a, 4, workspace, workspace_bytes, stream, "tg_kv_evict_f32");
}
int tg_kv_evict_f16(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::evict(a, 2, workspace, workspace_bytes, stream, "tg_kv_evict_f16");
}
int tg_kv_evict_bf16(const tg_kv_evict_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream) {
    return tg::evict(a, 2, workspace, workspace_bytes, stream, "tg_kv_evict_bf16");
}

}  // extern "C"
