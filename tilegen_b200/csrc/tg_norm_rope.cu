// Norms of queries and keys for each head, with the rotation in the same pass: forward
// (tg_norm_rope_*), on the way into the paged cache (tg_kv_append_normed_*) and the gradient
// (tg_norm_rope_backward_*).
//
// A head x of `dim` elements becomes y = R (r x w) with r = 1 / sqrt(mean(x^2) + eps), w = offset +
// weight and R the rotation at the token's position.  For the gradient dy of y, with g = R^T dy,
// u = g w and xh = r x:
//   dx = r (u - xh mean(u xh)),   dweight = sum of g xh over all rows of the tensor.
//
// * Bound: HBM, then issue slots.  A row is read once: a group of lanes holds it in registers, the sums
//   over it are shuffles, and the cosines and sines of a few tokens lie in shared memory for all heads of
//   q and k.  The gradient's two sums (x^2 and u x) are made in one round of shuffles.  16381 tokens of
//   32 and 8 heads of 128 in bfloat16, on several GPUs: forward (336 MB) 55 to 62 us, 5.4 to 6.1 TB/s,
//   78 % of issue slots; gradient (503 MB) 89 to 91 us, 5.5 to 5.7 TB/s; prompts into the cache (572 MB)
//   96 to 102 us, 5.6 to 6.0 TB/s (the measured copy: 6.5).
// * Rows come by cp.async into a ring of the thread's own places, three deep: in registers the rows ahead
//   cost the gradient its second CTA an SM (128 us without the ring) and the forward pass 11 of 66 us.
// * Statistics, rotation and sums are 32-bit, the angle 64-bit; each output is rounded once.  Where that
//   is to 16 bits, sine and cosine come from the special-function unit (2^-21 off).
// * The weights' gradients are summed by each thread over its rows, then over the CTA, then over the
//   CTAs by a second launch, always in the same order: calls are bit identical.
#include <algorithm>

#include "tg_rope.cuh"

namespace tg {
namespace {

constexpr int kNormDim = 256;  // longest head: eight elements a lane (16 in packs of eight)
constexpr int kRingDepth = 3;  // rows of a thread under way, and the one that is made
constexpr int kNormSmem = 112 * 1024;
enum { kForward, kAppend, kGradient };

template <typename T>
struct NormParams : NewTokens {
    // by kind: 0 q, 1 k, 2 v (append).  An output's row is page * out_page + slot * out_slot + head *
    // out_head; for q, and for k outside the append, the slot is the token and the page 0.
    const T* in[3];
    T* out[3];
    int64_t in_tok[3], in_head[3], out_page[3], out_slot[3], out_head[3];
    const T* grad[2];  // dy
    int64_t grad_tok[2], grad_head[2];
    int heads[3];
    const void* weight[2];
    int weight_f32[2], normed[2];
    float eps[2], offset[2];
    float* part;  // gradient: [CTA][kind][dim] sums
    // a step of a group's rows, `groups` further: tokens and heads, elements, and what comes on top where the
    // head's count wraps
    int step_tok[3], step_head[3];
    int64_t in_step[3], in_wrap[3], out_step[3], out_wrap[3], grad_step[2], grad_wrap[2];
    int dim, rot;
    const double* freq;
    float scale, sign;
    int acc_at;         // gradient: bytes in front of the threads' sums in shared memory
    int tile;           // tokens of a CTA, most tokens of its rounds (gradient)
    int chunks, lanes;  // items of a row, lanes of a row (a power of two)
};

__device__ __forceinline__ float weight_at(const void* w, int is_f32, const float*, int i) { return static_cast<const float*>(w)[i]; }
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int is_f32, const T*, int i) {
    return is_f32 ? static_cast<const float*>(w)[i] : to_f32(static_cast<const T*>(w)[i]);
}

// 1 / sqrt(v): within two units in the last place, exactly rounded where outputs have 32 bits.
template <typename T>
__device__ __forceinline__ float inverse_root(float v) {
    return sizeof(T) == 4 ? __frsqrt_rn(v) : rsqrtf(v);
}
// Two 32-bit numbers side by side: one instruction for both.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// VEC elements (a pack) are moved at once, 16 bytes where rows, strides and the parts of a row are
// multiples of that, else 8 bytes or single elements.  A lane has NI items of two packs of a row: the
// two halves of its pairs (HALF, or single elements of neighbouring pairs), or two packs of whole
// pairs or unturned elements, a stretch of the row apart so that the lanes' packs lie side by side.
// In registers an item is VEC pairs (a, b) either way, two of them in one 64-bit register: the packed
// instructions halve the arithmetic, which would otherwise take longer than the memory (16381 tokens
// of 40 heads of 128: 98 us with neither them nor the ring).
//
// LANES > 0: rows of exactly so many lanes with an item each that turns as a whole (heads of 64, 128 and
// 256 that rotate fully), so that sizes, places in shared memory and shuffles are known beforehand;
// else any row.
template <typename T, int VEC, bool HALF, int MODE, int LANES>
__global__ void __launch_bounds__(kRopeThreads, MODE == kGradient ? 2 : 4)
    norm_rope_kernel(const __grid_constant__ NormParams<T> p) {
    constexpr bool kFixed = LANES > 0;
    constexpr int NI = VEC >= 4 ? 1 : 4 / VEC;
    constexpr int NP = NI * VEC / 2;  // registers of pairs of a lane
    constexpr bool kApart = HALF || VEC == 1;       // a pair's elements are in different packs
    constexpr int kPairs = kApart ? VEC : VEC / 2;  // of a unit: an item (kApart) or a pack
    using P = Pack<T, VEC>;
    constexpr int kPack = VEC * (int)sizeof(T);  // bytes
    constexpr bool kRing = VEC > 1;
    constexpr int kDepth = kRingDepth, kRowPacks = NI * (MODE == kGradient ? 4 : 2);
    extern __shared__ __align__(16) unsigned char smem_bytes[];  // the ring; turns of [tile][pairs]; at the end the sums of the warps
    constexpr int s_ring = 0;
    float* const s_turn = reinterpret_cast<float*>(smem_bytes + (kRing ? kDepth * kRowPacks * kRopeThreads * kPack : 0));
    auto copy = [&](int to, const void* from) {
        if constexpr (kPack == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(smem_bytes) + to), "l"(from) : "memory");
        if constexpr (kPack == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(smem_bytes) + to), "l"(from) : "memory");
    };
    __shared__ __align__(16) float s_w[2][kNormDim];
    __shared__ double s_pos[kRopeTile];
    __shared__ int64_t s_page[kRopeTile], s_slot[kRopeTile];
    const int lanes = kFixed ? LANES : p.lanes, groups = kRopeThreads / lanes, chunks = kFixed ? LANES : p.chunks;
    const int dim = kFixed ? LANES * 2 * VEC : p.dim, rot = kFixed ? dim : p.rot;
    const int tid = threadIdx.x, lane = tid & (lanes - 1), group = tid / lanes;
    const int pairs = rot / 2, packs = dim / VEC;
    const int turning = kApart ? pairs / VEC : rot / VEC;  // units that turn
    const float inv_dim = 1.f / (float)dim;
    if constexpr (MODE == kGradient) pdl_trigger();

    // the packs of the lane's items, the same in every row
    int ia[NI], ib[NI];  // < 0: none
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = lane + i * lanes, rest = chunks - turning;
        if constexpr (kFixed) {
            ia[i] = c, ib[i] = c + chunks;
        } else if (c >= chunks) {
            ia[i] = ib[i] = -1;
        } else if (kApart && c < turning) {
            ia[i] = HALF ? c : 2 * c;
            ib[i] = HALF ? turning + c : 2 * c + 1;
        } else if (kApart) {
            ia[i] = turning + c;
            ib[i] = ia[i] + rest < packs ? ia[i] + rest : -1;
        } else {
            ia[i] = c;
            ib[i] = c + chunks < packs ? c + chunks : -1;
        }
    }

    // Weights in shared memory: four elements of a pack in one float4, those of all packs side by side
    // so that lanes read them without bank conflicts, in the order of the registers.
    auto weight_place = [&](int e) {
        if constexpr (VEC < 4) return e;
        const int pack = e / VEC, q = e % VEC / 4, j = e % 4;
        return (q * packs + pack) * 4 + (kApart ? j : (j & 1) * 2 + (j >> 1));
    };
    for (int i = tid; i < dim; i += kRopeThreads)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            s_w[k][weight_place(i)] =
                p.normed[k] && p.weight[k] ? p.offset[k] + weight_at(p.weight[k], p.weight_f32[k], (const T*)nullptr, i) : 1.f;
    // (the weights of a lane's pairs; of packs that it does not have, some)
    auto weights = [&](int kind, uint64_t (&wa)[NP], uint64_t (&wb)[NP]) {
        if constexpr (VEC >= 4) {
            const ulonglong2* w = reinterpret_cast<const ulonglong2*>(s_w[kind]);
            const int a = kFixed ? ia[0] : max(ia[0], 0), b = kFixed ? ib[0] : max(ib[0], 0);
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
                const ulonglong2 x = w[q * packs + a], y = w[q * packs + b];
                if constexpr (kApart) {
                    wa[2 * q] = x.x, wa[2 * q + 1] = x.y, wb[2 * q] = y.x, wb[2 * q + 1] = y.y;
                } else {
                    wa[q] = x.x, wb[q] = x.y, wa[NP / 2 + q] = y.x, wb[NP / 2 + q] = y.y;
                }
            }
        } else if constexpr (VEC == 2) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const float2 x = *reinterpret_cast<const float2*>(&s_w[kind][max(ia[i], 0) * 2]);
                const float2 y = *reinterpret_cast<const float2*>(&s_w[kind][max(ib[i], 0) * 2]);
                wa[i] = kApart ? two(x.x, x.y) : two(x.x, y.x), wb[i] = kApart ? two(y.x, y.y) : two(x.y, y.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; i += 2) {
                wa[i / 2] = two(s_w[kind][max(ia[i], 0)], s_w[kind][max(ia[i + 1], 0)]);
                wb[i / 2] = two(s_w[kind][max(ib[i], 0)], s_w[kind][max(ib[i + 1], 0)]);
            }
        }
    };
    // Packs to pairs and back.
    auto unpack = [&](const P (&x)[NI], const P (&y)[NI], uint64_t (&a)[NP], uint64_t (&b)[NP]) {
        float f[NI][VEC], g[NI][VEC];
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i].get(f[i]), y[i].get(g[i]);
        if constexpr (VEC == 1) {
#pragma unroll
            for (int i = 0; i < NI; i += 2) a[i / 2] = two(f[i][0], f[i + 1][0]), b[i / 2] = two(g[i][0], g[i + 1][0]);
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int m = 0; m < VEC / 2; ++m) {
                    const int at = i * VEC / 2 + m;
                    if constexpr (kApart) {
                        a[at] = two(f[i][2 * m], f[i][2 * m + 1]), b[at] = two(g[i][2 * m], g[i][2 * m + 1]);
                    } else if constexpr (VEC == 2) {
                        a[at] = two(f[i][0], g[i][0]), b[at] = two(f[i][1], g[i][1]);
                    } else {
                        const float* z = m < VEC / 4 ? f[i] + 4 * m : g[i] + 4 * m - VEC;
                        a[at] = two(z[0], z[2]), b[at] = two(z[1], z[3]);
                    }
                }
        }
    };
    auto repack = [&](const uint64_t (&a)[NP], const uint64_t (&b)[NP], P (&x)[NI], P (&y)[NI]) {
        float f[NI][VEC], g[NI][VEC];
        if constexpr (VEC == 1) {
#pragma unroll
            for (int i = 0; i < NI; i += 2) {
                const float2 u = both(a[i / 2]), v = both(b[i / 2]);
                f[i][0] = u.x, f[i + 1][0] = u.y, g[i][0] = v.x, g[i + 1][0] = v.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int m = 0; m < VEC / 2; ++m) {
                    const float2 u = both(a[i * VEC / 2 + m]), v = both(b[i * VEC / 2 + m]);
                    if constexpr (kApart) {
                        f[i][2 * m] = u.x, f[i][2 * m + 1] = u.y, g[i][2 * m] = v.x, g[i][2 * m + 1] = v.y;
                    } else if constexpr (VEC == 2) {
                        f[i][0] = u.x, g[i][0] = u.y, f[i][1] = v.x, g[i][1] = v.y;
                    } else {
                        float* z = m < VEC / 4 ? f[i] + 4 * m : g[i] + 4 * m - VEC;
                        z[0] = u.x, z[2] = u.y, z[1] = v.x, z[3] = v.y;
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i].put(f[i]), y[i].put(g[i]);
    };
    // Sum of u v over the lane's elements that are there.
    auto product = [&](const uint64_t (&ua)[NP], const uint64_t (&ub)[NP], const uint64_t (&va)[NP], const uint64_t (&vb)[NP]) {
        float sum = 0.f;
        if constexpr (VEC == 1) {
#pragma unroll
            for (int i = 0; i < NI; i += 2) {
                const float2 x = both(mul2(ua[i / 2], va[i / 2])), y = both(mul2(ub[i / 2], vb[i / 2]));
                sum += ((kFixed || ia[i] >= 0) ? x.x : 0.f) + ((kFixed || ia[i + 1] >= 0) ? x.y : 0.f);
                sum += ((kFixed || ib[i] >= 0) ? y.x : 0.f) + ((kFixed || ib[i + 1] >= 0) ? y.y : 0.f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                uint64_t sa = 0, sb = 0;  // of the item's two packs
#pragma unroll
                for (int m = 0; m < VEC / 2; ++m) {
                    const int at = i * VEC / 2 + m;
                    if constexpr (kApart) {
                        sa = fma2(ua[at], va[at], sa), sb = fma2(ub[at], vb[at], sb);
                    } else if constexpr (VEC == 2) {  // (pack a, pack b) in each register
                        sa = fma2(ua[at], va[at], sa), sa = fma2(ub[at], vb[at], sa);
                    } else if (m < VEC / 4) {
                        sa = fma2(ua[at], va[at], sa), sa = fma2(ub[at], vb[at], sa);
                    } else {
                        sb = fma2(ua[at], va[at], sb), sb = fma2(ub[at], vb[at], sb);
                    }
                }
                const float2 x = both(sa), y = both(sb);
                if constexpr (!kApart && VEC == 2) sum += ((kFixed || ia[i] >= 0) ? x.x : 0.f) + ((kFixed || ib[i] >= 0) ? x.y : 0.f);
                else sum += ((kFixed || ia[i] >= 0) ? x.x + x.y : 0.f) + ((kFixed || ib[i] >= 0) ? y.x + y.y : 0.f);
            }
        }
        return sum;
    };
    // Sines: of two pairs (cos, cos, sin, sin) in one float4, those of all units side by side; of units of
    // one pair (cos, sin).
    auto turn_place = [&](int pair) {
        const int unit = pair / kPairs, j = pair % kPairs;
        return kPairs == 1 ? 2 * unit : ((j >> 1) * turning + unit) * 4 + (j & 1);
    };
    auto turn2 = [&](uint64_t& a, uint64_t& b, ulonglong2 cs) {
        const uint64_t u = a, v = b, minus = mul2(cs.y, two(-1.f, -1.f));
        a = fma2(u, cs.x, mul2(v, minus));
        b = fma2(v, cs.x, mul2(u, cs.y));
    };
    auto rotate = [&](uint64_t (&a)[NP], uint64_t (&b)[NP], const float* turn) {
        if constexpr (kPairs == 1) {
            float f[2 * NP], g[2 * NP];
#pragma unroll
            for (int m = 0; m < NP; ++m) {
                const float2 u = both(a[m]), v = both(b[m]);
                f[2 * m] = u.x, f[2 * m + 1] = u.y, g[2 * m] = v.x, g[2 * m + 1] = v.y;
            }
#pragma unroll
            for (int j = 0; j < 2 * NP; ++j) {
                const int unit = VEC == 1 ? (ia[j % NI] < 0 ? turning : lane + j % NI * lanes) : (j & 1 ? ib[j / 2 % NI] : ia[j / 2 % NI]);
                if (unit < 0 || unit >= turning) continue;
                const float2 cs = *reinterpret_cast<const float2*>(turn + 2 * unit);
                const float u = f[j], v = g[j];
                f[j] = u * cs.x - v * cs.y;
                g[j] = v * cs.x + u * cs.y;
            }
#pragma unroll
            for (int m = 0; m < NP; ++m) a[m] = two(f[2 * m], f[2 * m + 1]), b[m] = two(g[2 * m], g[2 * m + 1]);
        } else {
            const ulonglong2* t = reinterpret_cast<const ulonglong2*>(turn);
            if constexpr (kApart) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int unit = lane + i * lanes;
                    if (!kFixed && unit >= turning) continue;
#pragma unroll
                    for (int q = 0; q < kPairs / 2; ++q) turn2(a[i * VEC / 2 + q], b[i * VEC / 2 + q], t[q * turning + unit]);
                }
            } else {
                if (kFixed || (ia[0] >= 0 && ia[0] < turning))
#pragma unroll
                    for (int q = 0; q < kPairs / 2; ++q) turn2(a[q], b[q], t[q * turning + ia[0]]);
                if (kFixed || (ib[0] >= 0 && ib[0] < turning))
#pragma unroll
                    for (int q = 0; q < kPairs / 2; ++q) turn2(a[NP / 2 + q], b[NP / 2 + q], t[q * turning + ib[0]]);
            }
        }
    };
    auto group_total = [&](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (lanes > o) v += __shfl_xor_sync(kFull, v, o);
        return v;
    };

    struct Row {
        P a[NI], b[NI];
        P ga[MODE == kGradient ? NI : 1], gb[MODE == kGradient ? NI : 1];
    };
    uint64_t acc_a[NP], acc_b[NP];
    int64_t t0;
    int tile;
    // A kind's rows of the tile: group g has rows g, g + groups, ...  Where the next row to load is.
    struct Walk {
        const T *in, *grad;
        int tt, h;  // token of the tile (>= tile: no row), head
    };
    auto begin = [&](int kind, Walk& w) {
        w.tt = group / p.heads[kind], w.h = group - w.tt * p.heads[kind];
        const int64_t t = t0 + w.tt;
        w.in = p.in[kind] + t * p.in_tok[kind] + w.h * p.in_head[kind];
        if constexpr (MODE == kGradient) w.grad = p.grad[kind] + t * p.grad_tok[kind] + w.h * p.grad_head[kind];
    };
    auto advance = [&](int kind, Walk& w) {
        w.tt += p.step_tok[kind], w.h += p.step_head[kind], w.in += p.in_step[kind];
        if constexpr (MODE == kGradient) w.grad += p.grad_step[kind];
        if (w.h >= p.heads[kind]) {
            w.h -= p.heads[kind], ++w.tt, w.in += p.in_wrap[kind];
            if constexpr (MODE == kGradient) w.grad += p.grad_wrap[kind];
        }
    };
    // Rows under way: in the thread's own places of a ring in shared memory (kRing), or in registers.
    auto ring_at = [&](int n, int pack) { return s_ring + ((n % kDepth * kRowPacks + pack) * kRopeThreads + tid) * kPack; };
    auto fetch = [&](const Walk& w, int n) {
        if (w.tt < tile) {
            const P *in = reinterpret_cast<const P*>(w.in), *g = reinterpret_cast<const P*>(w.grad);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                if ((kFixed || ia[i] >= 0)) copy(ring_at(n, 2 * i), in + ia[i]);
                if ((kFixed || ib[i] >= 0)) copy(ring_at(n, 2 * i + 1), in + ib[i]);
                if constexpr (MODE == kGradient) {
                    if ((kFixed || ia[i] >= 0)) copy(ring_at(n, 2 * NI + 2 * i), g + ia[i]);
                    if ((kFixed || ib[i] >= 0)) copy(ring_at(n, 2 * NI + 2 * i + 1), g + ib[i]);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto fetched = [&](int n, Row& x) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            x.a[i] = *reinterpret_cast<const P*>(smem_bytes + ring_at(n, 2 * i));
            x.b[i] = *reinterpret_cast<const P*>(smem_bytes + ring_at(n, 2 * i + 1));
            if constexpr (MODE == kGradient) {
                x.ga[i] = *reinterpret_cast<const P*>(smem_bytes + ring_at(n, 2 * NI + 2 * i));
                x.gb[i] = *reinterpret_cast<const P*>(smem_bytes + ring_at(n, 2 * NI + 2 * i + 1));
            }
        }
    };
    auto load = [&](const Walk& w, Row& x) {
        if (w.tt >= tile) return;
        const P *in = reinterpret_cast<const P*>(w.in), *g = reinterpret_cast<const P*>(w.grad);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if ((kFixed || ia[i] >= 0)) x.a[i] = in[ia[i]];
            if ((kFixed || ib[i] >= 0)) x.b[i] = in[ib[i]];
            if constexpr (MODE == kGradient) {
                if ((kFixed || ia[i] >= 0)) x.ga[i] = g[ia[i]];
                if ((kFixed || ib[i] >= 0)) x.gb[i] = g[ib[i]];
            }
        }
    };
    // The first rows of a kind, n0 rows after the tile's first.
    auto start = [&](int kind, Walk& w, Row& x, int n0) {
        begin(kind, w);
        if constexpr (kRing) {
            for (int d = 0; d < kDepth - 1; ++d) {
                fetch(w, n0 + d);
                advance(kind, w);
            }
        } else {
            load(w, x);
            advance(kind, w);
        }
    };
    // The tile's sines; its first rows are under way.
    auto sines_of_tile = [&] {
        __syncthreads();  // the tile before has read its own
        if constexpr (MODE == kAppend) {
            if (tid < tile) {
                const int64_t t = t0 + tid, at = slot_of_token(p, t, s_page[tid], s_slot[tid]);
                s_pos[tid] = (double)(p.positions ? p.positions[t] : p.position_base + at);
            }
            __syncthreads();
        }
        for (int i = tid; i < tile * pairs; i += kRopeThreads) {
            const int k = i / pairs, pair = i - k * pairs;
            const double pos = MODE == kAppend ? s_pos[k] : (double)p.positions[t0 + k];
            const float2 cs = turn_of<sizeof(T) == 2>(pos, p.freq[pair], p.scale, p.sign);
            float* to = s_turn + 2 * k * pairs + turn_place(pair);
            to[0] = cs.x;
            to[kPairs == 1 ? 1 : 2] = cs.y;
        }
        __syncthreads();
    };
    // All rows of a kind; its first are under way, and at the end those of kind `after` (< 0: none).
    auto rows_of = [&](int kind, int after, Walk& w, Row& x) {
        const int heads = p.heads[kind];
        const bool normed = kind < 2 && p.normed[kind];
        const bool paged = MODE == kAppend && kind > 0;
        const float eps = kind < 2 ? p.eps[kind] : 0.f;
        const int all = (tile * heads + groups - 1) / groups;  // the same for all lanes
        int tt = group / heads, h = group - tt * heads;        // of the row being made
        T* at = p.out[kind];
        if (!paged) at += (t0 + tt) * p.out_slot[kind] + h * p.out_head[kind];
        for (int n = 0; n < all; ++n) {
            Row y;
            if constexpr (kRing) {
                fetch(w, n + kDepth - 1);
                advance(kind, w);
                fetched(n, x);
            } else if (n + 1 < all) {
                load(w, y);
                advance(kind, w);
            }
            const bool there = tt < tile;
            P* out = reinterpret_cast<P*>(at);
            if (paged) {
                const int64_t page = there ? s_page[tt] : -1;
                if (page >= 0) out = reinterpret_cast<P*>(at + page * p.out_page[kind] + s_slot[tt] * p.out_slot[kind] + h * p.out_head[kind]);
                else out = nullptr;
            } else if (!there) {
                out = nullptr;
            }
            const float* turn = s_turn + 2 * tt * pairs;
            tt += p.step_tok[kind], h += p.step_head[kind];
            if (!paged) at += p.out_step[kind];
            if (h >= heads) {
                h -= heads, ++tt;
                if (!paged) at += p.out_wrap[kind];
            }
            if (MODE != kAppend || kind < 2) {  // values are copied as they are
                uint64_t a[NP], b[NP];
                unpack(x.a, x.b, a, b);
                if constexpr (MODE != kGradient) {
                    if (normed) {
                        const float r = inverse_root<T>(group_total(product(a, b, a, b)) * inv_dim + eps);
                        uint64_t wa[NP], wb[NP];
                        weights(kind, wa, wb);
#pragma unroll
                        for (int m = 0; m < NP; ++m) {
                            a[m] = mul2(a[m], mul2(two(r, r), wa[m]));
                            b[m] = mul2(b[m], mul2(two(r, r), wb[m]));
                        }
                    }
                    if (there) rotate(a, b, turn);
                    repack(a, b, x.a, x.b);
                } else {
                    uint64_t ga[NP], gb[NP];
                    unpack(x.ga, x.gb, ga, gb);
                    if (there) rotate(ga, gb, turn);
                    if (normed) {
                        uint64_t ua[NP], ub[NP];
                        weights(kind, ua, ub);
#pragma unroll
                        for (int m = 0; m < NP; ++m) ua[m] = mul2(ua[m], ga[m]), ub[m] = mul2(ub[m], gb[m]);
                        float ss = product(a, b, a, b), dot = product(ua, ub, a, b);
#pragma unroll
                        for (int o = 16; o; o >>= 1)
                            if (lanes > o) {
                                ss += __shfl_xor_sync(kFull, ss, o);
                                dot += __shfl_xor_sync(kFull, dot, o);
                            }
                        const float r = inverse_root<T>(ss * inv_dim + eps), m = -(dot * r * inv_dim);
                        const uint64_t r2 = two(r, r), m2 = two(m, m);
#pragma unroll
                        for (int k = 0; k < NP; ++k) {
                            const uint64_t xa = mul2(a[k], r2), xb = mul2(b[k], r2);
                            if (there) {
                                acc_a[k] = fma2(ga[k], xa, acc_a[k]);
                                acc_b[k] = fma2(gb[k], xb, acc_b[k]);
                            }
                            ga[k] = mul2(r2, fma2(xa, m2, ua[k]));
                            gb[k] = mul2(r2, fma2(xb, m2, ub[k]));
                        }
                    }
                    repack(ga, gb, x.a, x.b);
                }
            }
            if (out) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if ((kFixed || ia[i] >= 0)) out[ia[i]] = x.a[i];
                    if ((kFixed || ib[i] >= 0)) out[ib[i]] = x.b[i];
                }
            }
            if constexpr (!kRing) x = y;
        }
        if constexpr (kRing) asm volatile("cp.async.wait_group 0;" ::: "memory");  // (of no rows)
        if (after >= 0) start(after, w, x, 0);
    };

    if constexpr (MODE != kGradient) {
        // a tile of tokens a CTA
        t0 = (int64_t)blockIdx.x * p.tile;
        tile = (int)min((int64_t)p.tile, p.tokens - t0);
        constexpr int kKinds = MODE == kAppend ? 3 : 2;
        auto from = [&](int kind) {  // the first kind from there on that has heads
            while (kind < kKinds && p.heads[kind] == 0) ++kind;
            return kind < kKinds ? kind : -1;
        };
        Walk w;
        Row x;
        int kind = from(0);
        start(kind, w, x, 0);
        sines_of_tile();
#pragma unroll 1
        while (kind >= 0) {
            const int after = from(kind + 1);
            rows_of(kind, after, w, x);
            kind = after;
        }
    } else {
        float* const s_sum = s_turn;  // [warp][dim]
        constexpr int kWarps = kRopeThreads / 32;
        const int warp = tid >> 5;
        const int64_t share = p.tokens * (blockIdx.x + 1) / gridDim.x;  // my tokens end here
        // A thread's sums are kept in shared memory between the tiles, those of one kind at a time in
        // registers: both together would not fit.
        ulonglong2* const s_acc = reinterpret_cast<ulonglong2*>(smem_bytes + p.acc_at) + tid;  // [kind][NP][thread]
#pragma unroll
        for (int m = 0; m < 2 * NP; ++m) s_acc[m * kRopeThreads] = make_ulonglong2(0, 0);
        const int kind0 = p.heads[0] > 0 ? 0 : 1, kind1 = p.heads[1] > 0 ? 2 : 1;
        for (t0 = p.tokens * blockIdx.x / gridDim.x; t0 < share; t0 += p.tile) {
            tile = (int)min((int64_t)p.tile, share - t0);
            Walk w;
            Row x;
            start(kind0, w, x, 0);
            sines_of_tile();
#pragma unroll 1
            for (int kind = kind0; kind < kind1; ++kind) {
#pragma unroll
                for (int m = 0; m < NP; ++m) acc_a[m] = acc_b[m] = 0;
                rows_of(kind, kind + 1 < kind1 ? kind + 1 : -1, w, x);
#pragma unroll
                for (int m = 0; m < NP; ++m) {
                    ulonglong2& at = s_acc[(kind * NP + m) * kRopeThreads];
                    const ulonglong2 v = at;
                    at = make_ulonglong2(add2(v.x, acc_a[m]), add2(v.y, acc_b[m]));
                }
            }
        }
#pragma unroll 1
        for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
            for (int m = 0; m < NP; ++m) {
                const ulonglong2 v = s_acc[(kind * NP + m) * kRopeThreads];
                acc_a[m] = v.x, acc_b[m] = v.y;
            }
            // the groups of a warp, then the warps one after the other
            __syncthreads();
            float f[NP * 2], g[NP * 2];
#pragma unroll
            for (int m = 0; m < NP; ++m) {
                const float2 u = both(acc_a[m]), v = both(acc_b[m]);
                f[2 * m] = u.x, f[2 * m + 1] = u.y, g[2 * m] = v.x, g[2 * m + 1] = v.y;
            }
#pragma unroll
            for (int j = 0; j < NP * 2; ++j)
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    float v = side ? g[j] : f[j];
#pragma unroll
                    for (int o = 16; o; o >>= 1)
                        if (o >= lanes) v += __shfl_xor_sync(kFull, v, o);
                    // the element of pair j
                    int e;
                    if constexpr (kApart) {
                        const int pack = side ? ib[j / VEC] : ia[j / VEC];
                        e = pack < 0 ? -1 : pack * VEC + j % VEC;
                    } else {
                        const bool second = j % VEC >= VEC / 2;
                        const int pack = second ? ib[j / VEC] : ia[j / VEC];
                        e = pack < 0 ? -1 : pack * VEC + 2 * (j % VEC - (second ? VEC / 2 : 0)) + side;
                    }
                    if ((tid & 31) < lanes && e >= 0) s_sum[warp * dim + e] = v;
                }
            __syncthreads();
            for (int i = tid; i < dim; i += kRopeThreads) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) v += s_sum[k * dim + i];
                p.part[((int64_t)blockIdx.x * 2 + kind) * dim + i] = v;
            }
            __syncthreads();
        }
    }
}

constexpr int kSumCols = 32, kSumRows = 32;

// dweight of a kind (blockIdx.y): the CTAs' sums, 32 interleaved runs of them first (with eight runs of 37
// loads one after the other this took 10 of the gradient's 90 us).
template <typename T>
__global__ void __launch_bounds__(kSumCols* kSumRows) weight_sum_kernel(const float* part, int ctas, int dim, void* dq, void* dk,
                                                                        int q_f32, int k_f32) {
    __shared__ float s[kSumRows][kSumCols];
    pdl_wait();
    const int k = blockIdx.y, x = threadIdx.x % kSumCols, y = threadIdx.x / kSumCols, i = blockIdx.x * kSumCols + x;
    void* const out = k ? dk : dq;
    if (!out) return;
    float v = 0.f;
    if (i < dim)
#pragma unroll 10
        for (int c = y; c < ctas; c += kSumRows) v += part[((int64_t)c * 2 + k) * dim + i];
    s[y][x] = v;
    __syncthreads();
    if (y == 0 && i < dim) {
#pragma unroll
        for (int r = 1; r < kSumRows; ++r) v += s[r][x];
        if (k ? k_f32 : q_f32) static_cast<float*>(out)[i] = v;
        else static_cast<T*>(out)[i] = from_f32<T>(v);
    }
}

// CTAs of the gradient: two on each SM (its registers), no more than tokens.
int gradient_ctas(int64_t tokens) { return (int)std::min<int64_t>(tokens, 2 * kSMs); }

// Tokens of a CTA: enough that each group of lanes has a few rows for its share of the sines, but at
// least eight CTAs an SM (a few tokens are one CTA each).
int tile_of(int64_t tokens, int rows, int groups, int pairs) {
    int64_t tile = ceil_div(8ll * groups, std::max(rows, 1));
    tile = std::min<int64_t>({tile, kRopeTile, std::max<int64_t>(1, tokens / (kSMs * 8)),
                              pairs ? std::max<int64_t>(1, kRopeSmem / (pairs * 8)) : kRopeTile});
    return (int)tile;
}

template <typename T>
struct Shape {
    int vec, chunks, lanes, groups;
};

// How rows are moved: by the or of all addresses and strides in bytes.
template <typename T>
Shape<T> shape_of(uint64_t all, int dim, int rot, bool half) {
    Shape<T> s;
    for (s.vec = 16 / (int)sizeof(T); s.vec > 1; s.vec = s.vec * (int)sizeof(T) == 16 ? s.vec / 2 : 1)
        if (all % (s.vec * sizeof(T)) == 0 && dim % s.vec == 0 && rot % (half ? 2 * s.vec : s.vec) == 0) break;
    s.chunks = half || s.vec == 1 ? rot / 2 / s.vec + ((dim - rot) / s.vec + 1) / 2 : (dim / s.vec + 1) / 2;
    const int items = s.vec >= 4 ? 1 : 4 / s.vec;
    for (s.lanes = 1; s.lanes * items < s.chunks;) s.lanes *= 2;
    s.groups = kRopeThreads / s.lanes;
    return s;
}

template <typename T>
struct NormKernel {
    void (*run)(NormParams<T>);
    SmemOnce* once;
};
template <typename T, int VEC, bool HALF, int MODE, int LANES>
NormKernel<T> norm_kernel_of() {
    static SmemOnce once;
    return {norm_rope_kernel<T, VEC, HALF, MODE, LANES>, &once};
}
// The kernel for packs of vec elements and, where every lane has an item that turns, rows of `lanes`.
template <typename T, int WIDE, bool HALF, int MODE>
NormKernel<T> norm_kernel(int vec, int lanes) {
    if (vec == WIDE / 2) return norm_kernel_of<T, WIDE / 2, HALF, MODE, 0>();
    if (vec == 1) return norm_kernel_of<T, 1, HALF, MODE, 0>();
    constexpr int kOne = 64 / (2 * WIDE);  // lanes of heads of 64
    return lanes == kOne       ? norm_kernel_of<T, WIDE, HALF, MODE, kOne>()
           : lanes == 2 * kOne ? norm_kernel_of<T, WIDE, HALF, MODE, 2 * kOne>()
           : lanes == 4 * kOne ? norm_kernel_of<T, WIDE, HALF, MODE, 4 * kOne>()
                               : norm_kernel_of<T, WIDE, HALF, MODE, 0>();
}

// Fits p to the rows and launches it.
template <typename T, int MODE>
int run(NormParams<T>& p, int layout, int& ctas, cudaStream_t st, const char* what) {
    const bool half = layout == TG_ROPE_HALF;
    uint64_t all = 0;
    for (int k = 0; k < 3; ++k) {
        if (p.heads[k] == 0) continue;
        all |= reinterpret_cast<uint64_t>(p.in[k]) | reinterpret_cast<uint64_t>(p.out[k]);
        all |= (uint64_t)(p.in_tok[k] | p.in_head[k] | p.out_page[k] | p.out_slot[k] | p.out_head[k]) * sizeof(T);
        if (MODE == kGradient && k < 2)
            all |= reinterpret_cast<uint64_t>(p.grad[k]) | (uint64_t)(p.grad_tok[k] | p.grad_head[k]) * sizeof(T);
    }
    const int rows = p.heads[0] + p.heads[1] + p.heads[2];
    const Shape<T> s = shape_of<T>(all, p.dim, p.rot, half);
    p.chunks = s.chunks, p.lanes = s.lanes;
    for (int k = 0; k < 3; ++k) {
        if (p.heads[k] == 0) continue;
        const int64_t n = p.heads[k], dt = s.groups / n, dh = s.groups - dt * n;
        p.step_tok[k] = (int)dt, p.step_head[k] = (int)dh;
        p.in_step[k] = dt * p.in_tok[k] + dh * p.in_head[k], p.in_wrap[k] = p.in_tok[k] - n * p.in_head[k];
        p.out_step[k] = dt * p.out_slot[k] + dh * p.out_head[k], p.out_wrap[k] = p.out_slot[k] - n * p.out_head[k];
        if (MODE == kGradient && k < 2)
            p.grad_step[k] = dt * p.grad_tok[k] + dh * p.grad_head[k], p.grad_wrap[k] = p.grad_tok[k] - n * p.grad_head[k];
    }
    const int pairs = p.rot / 2;
    const int packs = (s.vec >= 4 ? 1 : 4 / s.vec) * (MODE == kGradient ? 4 : 2);  // of a thread's row
    if (MODE == kGradient) {
        ctas = gradient_ctas(p.tokens);
        p.tile = (int)std::min<int64_t>({kRopeTile, ceil_div(p.tokens, ctas), std::max(1, kRopeSmem / 2 / (std::max(pairs, 1) * 8))});
    } else {
        p.tile = tile_of(p.tokens, rows, MODE == kAppend ? 2 * s.groups : s.groups, pairs);
        ctas = (int)ceil_div(p.tokens, p.tile);
    }
    size_t smem = (size_t)p.tile * pairs * sizeof(float2);
    if (MODE == kGradient) smem = std::max(smem, (size_t)(kRopeThreads / 32) * p.dim * sizeof(float));
    constexpr int WIDE = 16 / (int)sizeof(T);
    if (s.vec > 1) smem += (size_t)kRingDepth * packs * kRopeThreads * s.vec * sizeof(T);
    if (MODE == kGradient) {
        smem = (smem + 15) / 16 * 16;
        p.acc_at = (int)smem;
        smem += (size_t)2 * (packs / 4 * s.vec / 2) * kRopeThreads * 16;
    }
    const bool full = s.vec == WIDE && p.rot == p.dim && s.chunks == s.lanes && p.dim == s.lanes * 2 * WIDE;
    auto kernel = half ? norm_kernel<T, WIDE, true, MODE>(s.vec, full ? s.lanes : 0) : norm_kernel<T, WIDE, false, MODE>(s.vec, full ? s.lanes : 0);
    if (smem > 40 * 1024) {  // (with what is declared, past 48 KB)
        const int rc = kernel.once->raise(reinterpret_cast<const void*>(kernel.run), kNormSmem);
        if (rc != TG_OK) return rc;
    }
    kernel.run<<<(unsigned)ctas, kRopeThreads, smem, st>>>(p);
    return check_launch(what);
}

template <typename T>
int set_norm(NormParams<T>& p, int kind, const tg_head_norm* n, const char* op) {
    p.normed[kind] = n != nullptr;
    if (!n) return TG_OK;
    if (!(n->eps >= 0.0)) return set_error(TG_EINVAL, "%s: eps must not be negative (got %g)", op, n->eps);
    p.weight[kind] = n->weight, p.weight_f32[kind] = n->weight_f32 != 0;
    p.eps[kind] = (float)n->eps, p.offset[kind] = (float)n->offset;
    return TG_OK;
}

int check_heads(int64_t tokens, int32_t dim, int32_t q_heads, int32_t k_heads, const tg_rope* r, const int64_t* positions,
                const char* op) {
    if (tokens < 0 || tokens > INT32_MAX || dim < 1 || q_heads < 0 || k_heads < 0)
        return set_error(TG_EINVAL, "%s: bad size (tokens=%lld dim=%d heads=%d, %d)", op, (long long)tokens, dim, q_heads, k_heads);
    if (dim > kNormDim) return set_error(TG_EUNSUPPORTED, "%s: heads of more than %d elements (got %d)", op, kNormDim, dim);
    // rows of a round are counted in 32 bits
    if ((int64_t)q_heads + k_heads > (1 << 24)) return set_error(TG_EUNSUPPORTED, "%s: more than 2^24 heads", op);
    if (!r) return TG_OK;
    const int rc = check_rope(r, dim, op);
    if (rc == TG_OK && r->rot_dim > 0 && tokens > 0 && !positions) return set_error(TG_EINVAL, "%s: null positions", op);
    return rc;
}

template <typename T>
void set_rope(NormParams<T>& p, const tg_rope* r, float sign) {
    p.sign = sign;
    if (r) p.rot = r->rot_dim, p.freq = r->freq, p.scale = (float)r->scale;
}

template <typename T>
int norm_rope(const tg_norm_rope_args* a, tg_stream_t stream, const char* op) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_heads(a->tokens, a->dim, a->q_heads, a->k_heads, a->rope, a->positions, op);
    NormParams<T> p = {};
    if (rc == TG_OK) rc = set_norm(p, 0, a->q_norm, op);
    if (rc == TG_OK) rc = set_norm(p, 1, a->k_norm, op);
    if (rc != TG_OK) return rc;
    if (a->flags) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if (a->tokens == 0 || a->q_heads + a->k_heads == 0) return TG_OK;
    const tg_rows* in[2] = {&a->q, &a->k};
    const tg_rows* out[2] = {&a->q_out, &a->k_out};
    p.heads[0] = a->q_heads, p.heads[1] = a->k_heads;
    for (int k = 0; k < 2; ++k) {
        if (p.heads[k] == 0) continue;
        if (!in[k]->data || !out[k]->data) return set_error(TG_EINVAL, "%s: null %s", op, k ? "k/k_out" : "q/q_out");
        p.in[k] = static_cast<const T*>(in[k]->data), p.out[k] = static_cast<T*>(out[k]->data);
        p.in_tok[k] = stride_of(a->tokens, in[k]->token_stride), p.in_head[k] = stride_of(p.heads[k], in[k]->head_stride);
        p.out_slot[k] = stride_of(a->tokens, out[k]->token_stride), p.out_head[k] = stride_of(p.heads[k], out[k]->head_stride);
    }
    p.tokens = a->tokens, p.positions = a->positions, p.dim = a->dim;
    set_rope(p, a->rope, 1.f);
    int ctas;
    return run<T, kForward>(p, a->rope ? a->rope->layout : TG_ROPE_HALF, ctas, static_cast<cudaStream_t>(stream), op);
}

template <typename T>
int append(const tg_kv_append_args* a, const tg_head_norm* q_norm, const tg_head_norm* k_norm, tg_stream_t stream, const char* op) {
    bool done;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    NormParams<T> p = {};
    int rc = set_norm(p, 0, q_norm, op);
    if (rc == TG_OK) rc = set_norm(p, 1, k_norm, op);
    if (rc == TG_OK && a && a->cache && a->cache->dim > kNormDim)
        rc = set_error(TG_EUNSUPPORTED, "%s: heads of more than %d elements (got %d)", op, kNormDim, a->cache->dim);
    if (rc == TG_OK) rc = check_append(a, op, st, done);
    if (rc != TG_OK || done) return rc;
    const tg_paged_kv& c = *a->cache;
    const tg_rows* in[3] = {a->q, &a->k, &a->v};
    if (a->q && a->q_heads > 0) {
        p.heads[0] = a->q_heads;
        p.out[0] = static_cast<T*>(a->q_out->data);
        p.out_slot[0] = stride_of(a->tokens, a->q_out->token_stride), p.out_head[0] = stride_of(a->q_heads, a->q_out->head_stride);
    }
    p.heads[1] = p.heads[2] = c.heads;
    if ((int64_t)p.heads[0] + 2ll * c.heads > (1 << 24)) return set_error(TG_EUNSUPPORTED, "%s: more than 2^24 heads", op);
    p.out[1] = static_cast<T*>(c.k), p.out[2] = static_cast<T*>(c.v);
    p.out_page[1] = stride_of(c.pages, c.k_page_stride), p.out_page[2] = stride_of(c.pages, c.v_page_stride);
    p.out_slot[1] = stride_of(c.page_size, c.k_slot_stride), p.out_slot[2] = stride_of(c.page_size, c.v_slot_stride);
    p.out_head[1] = stride_of(c.heads, c.k_head_stride), p.out_head[2] = stride_of(c.heads, c.v_head_stride);
    for (int k = 0; k < 3; ++k) {
        if (p.heads[k] == 0) continue;
        p.in[k] = static_cast<const T*>(in[k]->data);
        p.in_tok[k] = stride_of(a->tokens, in[k]->token_stride), p.in_head[k] = stride_of(p.heads[k], in[k]->head_stride);
    }
    p.dim = c.dim;
    set_rope(p, a->rope, 1.f);
    new_tokens(*a, p);
    int ctas;
    return run<T, kAppend>(p, a->rope ? a->rope->layout : TG_ROPE_HALF, ctas, st, op);
}

// Bytes of the CTAs' sums, for any rounds: at most two CTAs an SM.
size_t gradient_bytes(const tg_norm_rope_grad_args* a) {
    if (!a || a->tokens <= 0 || a->dim < 1 || a->dim > kNormDim) return 0;
    return (size_t)gradient_ctas(a->tokens) * 2 * a->dim * sizeof(float);
}

template <typename T>
int backward(const tg_norm_rope_grad_args* a, void* workspace, size_t workspace_bytes, tg_stream_t stream, const char* op) {
    if (!a) return set_error(TG_EINVAL, "%s: null arguments", op);
    int rc = check_heads(a->tokens, a->dim, a->q_heads, a->k_heads, a->rope, a->positions, op);
    NormParams<T> p = {};
    if (rc == TG_OK) rc = set_norm(p, 0, a->q_norm, op);
    if (rc == TG_OK) rc = set_norm(p, 1, a->k_norm, op);
    if (rc != TG_OK) return rc;
    if (a->flags) return set_error(TG_EINVAL, "%s: unknown flags 0x%x", op, a->flags);
    if ((a->dq_weight && !a->q_norm) || (a->dk_weight && !a->k_norm))
        return set_error(TG_EINVAL, "%s: a weight's gradient without its norm", op);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const tg_rows* in[2] = {&a->q, &a->k};
    const tg_rows* grad[2] = {&a->dq_out, &a->dk_out};
    const tg_rows* out[2] = {&a->dq, &a->dk};
    p.heads[0] = a->q_heads, p.heads[1] = a->k_heads;
    for (int k = 0; k < 2; ++k) {
        if (p.heads[k] == 0 || a->tokens == 0) continue;
        if (!in[k]->data || !out[k]->data || !grad[k]->data)
            return set_error(TG_EINVAL, "%s: null %s", op, k ? "k/dk_out/dk" : "q/dq_out/dq");
        p.in[k] = static_cast<const T*>(in[k]->data), p.out[k] = static_cast<T*>(out[k]->data);
        p.grad[k] = static_cast<const T*>(grad[k]->data);
        p.in_tok[k] = stride_of(a->tokens, in[k]->token_stride), p.in_head[k] = stride_of(p.heads[k], in[k]->head_stride);
        p.out_slot[k] = stride_of(a->tokens, out[k]->token_stride), p.out_head[k] = stride_of(p.heads[k], out[k]->head_stride);
        p.grad_tok[k] = stride_of(a->tokens, grad[k]->token_stride), p.grad_head[k] = stride_of(p.heads[k], grad[k]->head_stride);
    }
    p.tokens = a->tokens, p.positions = a->positions, p.dim = a->dim;
    set_rope(p, a->rope, -1.f);
    int ctas = 0;  // no rows: the weights' gradients are zeros
    if (a->tokens > 0 && a->q_heads + a->k_heads > 0) {
        const size_t need = gradient_bytes(a);
        if (!workspace || workspace_bytes < need)
            return set_error(TG_ENOMEM, "%s: workspace of %zu bytes needed (got %zu)", op, need, workspace_bytes);
        if (reinterpret_cast<uintptr_t>(workspace) % 16) return set_error(TG_EINVAL, "%s: the workspace must be 16-byte aligned", op);
        p.part = static_cast<float*>(workspace);
        rc = run<T, kGradient>(p, a->rope ? a->rope->layout : TG_ROPE_HALF, ctas, st, op);
        if (rc != TG_OK) return rc;
    }
    if (!a->dq_weight && !a->dk_weight) return TG_OK;
    return launch_pdl(op, weight_sum_kernel<T>, dim3((unsigned)ceil_div(a->dim, kSumCols), 2), kSumCols * kSumRows, 0, st,
                      static_cast<const float*>(workspace), ctas, a->dim, a->dq_weight, a->dk_weight, p.weight_f32[0], p.weight_f32[1]);
}

}  // namespace
}  // namespace tg

extern "C" {

size_t tg_norm_rope_backward_workspace_bytes(const tg_norm_rope_grad_args* a) { return tg::gradient_bytes(a); }

#define TG_NORM_ENTRY(SUFFIX, T)                                                                                       \
    int tg_norm_rope_##SUFFIX(const tg_norm_rope_args* a, tg_stream_t stream) {                                        \
        return tg::norm_rope<T>(a, stream, "tg_norm_rope_" #SUFFIX);                                                   \
    }                                                                                                                  \
    int tg_kv_append_normed_##SUFFIX(const tg_kv_append_args* a, const tg_head_norm* q_norm, const tg_head_norm* k_norm, \
                                     tg_stream_t stream) {                                                             \
        return tg::append<T>(a, q_norm, k_norm, stream, "tg_kv_append_normed_" #SUFFIX);                               \
    }                                                                                                                  \
    int tg_norm_rope_backward_##SUFFIX(const tg_norm_rope_grad_args* a, void* workspace, size_t workspace_bytes,       \
                                       tg_stream_t stream) {                                                           \
        return tg::backward<T>(a, workspace, workspace_bytes, stream, "tg_norm_rope_backward_" #SUFFIX);               \
    }
TG_NORM_ENTRY(f32, float)
TG_NORM_ENTRY(f16, __half)
TG_NORM_ENTRY(bf16, __nv_bfloat16)

}  // extern "C"
