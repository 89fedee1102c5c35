// Norms of queries and keys for each head, with the rotation in the same pass: forward
// (tg_norm_rope_*), on the way into the paged cache (tg_kv_append_normed_*) and the gradient
// (tg_norm_rope_backward_*).
//
// A head x of `dim` elements becomes y = R (r x w) with r = 1 / sqrt(mean(x^2) + eps), w = offset +
// weight and R the rotation at the token's position.  For the gradient dy of y, with g = R^T dy,
// u = g w and xh = r x:
//   dx = r (u - xh mean(u xh)),   dweight = sum of g xh over all rows of the tensor.
//
// * A row is read once: a group of lanes holds it in registers, the sums over it are shuffles, and
//   the cosines and sines of a few tokens lie in shared memory for all heads of q and k.  The
//   gradient's two sums (x^2 and u x) are made in one round of shuffles.
// * Statistics, rotation and sums are 32-bit, the angle 64-bit; each output is rounded once.
// * The weights' gradients are summed by each thread over its rows, then over the CTA, then over the
//   CTAs by a second launch, always in the same order: calls are bit identical.
#include <algorithm>

#include "tg_rope.cuh"

namespace tg {
namespace {

constexpr int kNormDim = 256;  // longest head: eight elements a lane (16 in packs of eight)
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
    int dim, rot;
    const double* freq;
    float scale, sign;
    int tile;                   // tokens of a round
    int chunks, lanes, groups;  // items of a row, lanes of a row (a power of two), rows of a CTA at a time
};

__device__ __forceinline__ float weight_at(const void* w, int is_f32, const float*, int i) { return static_cast<const float*>(w)[i]; }
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int is_f32, const T*, int i) {
    return is_f32 ? static_cast<const float*>(w)[i] : to_f32(static_cast<const T*>(w)[i]);
}

// VEC elements (a pack) are moved at once, 16 bytes where rows, strides and the parts of a row are
// multiples of that, else 8 bytes or single elements.  A lane has NI items of two packs of a row: the
// two halves of its pairs (HALF, or single elements of neighbouring pairs), or two packs of whole
// pairs or unturned elements, a stretch of the row apart so that the lanes' packs lie side by side.
template <typename T, int VEC, bool HALF, int MODE>
__global__ void __launch_bounds__(kRopeThreads, MODE == kGradient ? 2 : 3) norm_rope_kernel(const __grid_constant__ NormParams<T> p) {
    constexpr int NI = VEC >= 4 ? 1 : 4 / VEC;
    constexpr bool kApart = HALF || VEC == 1;
    constexpr int kPairs = kApart ? VEC : VEC / 2;  // of an item's pack
    constexpr int kKinds = MODE == kAppend ? 3 : 2;
    using P = Pack<T, VEC>;
    extern __shared__ float4 s_turn4[];  // (cos, sin) of [tile][pairs]; at the end the sums of the warps
    float2* const s_turn = reinterpret_cast<float2*>(s_turn4);
    __shared__ __align__(16) float s_w[2][kNormDim];
    __shared__ double s_pos[kRopeTile];
    __shared__ int64_t s_page[kRopeTile], s_slot[kRopeTile];
    const int tid = threadIdx.x, lane = tid & (p.lanes - 1), group = tid / p.lanes;
    const int pairs = p.rot / 2, packs = p.dim / VEC;
    const int turning = kApart ? pairs / VEC : p.rot / VEC;  // packs (or pairs of packs) that turn
    const float inv_dim = 1.f / (float)p.dim;
    const int64_t rounds = (p.tokens + p.tile - 1) / p.tile;
    if constexpr (MODE == kGradient) pdl_trigger();

    // the packs of the lane's items, the same in every row
    int ia[NI], ib[NI];  // < 0: none
    bool turns[NI];      // kApart: the item's pairs turn
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = lane + i * p.lanes, rest = p.chunks - turning;
        turns[i] = false;
        if (c >= p.chunks) {
            ia[i] = ib[i] = -1;
        } else if (kApart && c < turning) {
            ia[i] = HALF ? c : 2 * c;
            ib[i] = HALF ? turning + c : 2 * c + 1;
            turns[i] = true;
        } else if (kApart) {
            ia[i] = turning + c;
            ib[i] = ia[i] + rest < packs ? ia[i] + rest : -1;
        } else {
            ia[i] = c;
            ib[i] = c + p.chunks < packs ? c + p.chunks : -1;
        }
    }
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
    auto rotate = [&](float (&a)[NI][VEC], float (&b)[NI][VEC], const float2* turn) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            float2 cs[kPairs];
            if constexpr (kApart) {
                if (!turns[i]) continue;
                sines(turn, HALF ? ia[i] : ia[i] / 2, cs);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = a[i][j], w = b[i][j];
                    a[i][j] = u * cs[j].x - w * cs[j].y;
                    b[i][j] = w * cs[j].x + u * cs[j].y;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int at = k ? ib[i] : ia[i];
                    float(&f)[VEC] = k ? b[i] : a[i];
                    if (at < 0 || at >= turning) continue;
                    sines(turn, at, cs);
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) {
                        const float u = f[2 * j], w = f[2 * j + 1];
                        f[2 * j] = u * cs[j].x - w * cs[j].y;
                        f[2 * j + 1] = w * cs[j].x + u * cs[j].y;
                    }
                }
            }
        }
    };

    for (int i = tid; i < p.dim; i += kRopeThreads)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            s_w[k][i] = p.normed[k] && p.weight[k] ? p.offset[k] + weight_at(p.weight[k], p.weight_f32[k], (const T*)nullptr, i) : 1.f;
    float acc[MODE == kGradient ? 2 : 1][NI][2][VEC] = {};

    for (int64_t round = blockIdx.x; round < rounds; round += gridDim.x) {
        const int64_t t0 = round * p.tile;
        const int tile = (int)min((int64_t)p.tile, p.tokens - t0);
        __syncthreads();  // the round before has read its sines
        if (tid < tile) {
            const int64_t t = t0 + tid;
            if constexpr (MODE == kAppend) {
                const int64_t at = slot_of_token(p, t, s_page[tid], s_slot[tid]);
                s_pos[tid] = (double)(p.positions ? p.positions[t] : p.position_base + at);
            } else if (pairs) {
                s_pos[tid] = (double)p.positions[t];
            }
        }
        __syncthreads();
        for (int i = tid; i < tile * pairs; i += kRopeThreads) {
            const int k = i / pairs, pair = i - k * pairs;
            s_turn[k * pairs + place(pair / kPairs, pair % kPairs)] = turn_of(s_pos[k], p.freq[pair], p.scale, p.sign);
        }
        __syncthreads();

        auto rows_of = [&](auto kind_) {
            constexpr int kind = decltype(kind_)::value;
            const int heads = p.heads[kind], rows = tile * heads;
            if (rows == 0) return;
            const int dt = p.groups / heads, dh = p.groups - dt * heads;
            struct Row {
                P a[NI], b[NI];
                P ga[MODE == kGradient ? NI : 1], gb[MODE == kGradient ? NI : 1];
                T* out;
                int tt;
            };
            int tt = group / heads, h = group - tt * heads;
            // the lane's next row, its loads under way
            auto next = [&](Row& x) {
                x.out = nullptr;
                x.tt = tt;
                if (tt < tile) {
                    const int64_t t = t0 + tt;
                    int64_t page = 0, slot = t;
                    if (MODE == kAppend && kind > 0) page = s_page[tt], slot = s_slot[tt];
                    if (page >= 0) {
                        const P* in = reinterpret_cast<const P*>(p.in[kind] + t * p.in_tok[kind] + h * p.in_head[kind]);
                        x.out = p.out[kind] + page * p.out_page[kind] + slot * p.out_slot[kind] + h * p.out_head[kind];
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            if (ia[i] >= 0) x.a[i] = in[ia[i]];
                            if (ib[i] >= 0) x.b[i] = in[ib[i]];
                        }
                        if constexpr (MODE == kGradient) {
                            const P* g = reinterpret_cast<const P*>(p.grad[kind] + t * p.grad_tok[kind] + h * p.grad_head[kind]);
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                if (ia[i] >= 0) x.ga[i] = g[ia[i]];
                                if (ib[i] >= 0) x.gb[i] = g[ib[i]];
                            }
                        }
                    }
                }
                tt += dt;
                h += dh;
                if (h >= heads) h -= heads, ++tt;
            };
            auto store = [&](Row& x) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (ia[i] >= 0) reinterpret_cast<P*>(x.out)[ia[i]] = x.a[i];
                    if (ib[i] >= 0) reinterpret_cast<P*>(x.out)[ib[i]] = x.b[i];
                }
            };
            const int turnsOf = (rows + p.groups - 1) / p.groups;  // rounds of the groups, the same for all lanes
            Row x;
            next(x);
            if constexpr (kind == 2) {  // values are copied as they are
                for (int n = 0; n < turnsOf; ++n) {
                    Row y;
                    if (n + 1 < turnsOf) next(y);
                    if (x.out) store(x);
                    x = y;
                }
                return;
            } else {
                const bool normed = p.normed[kind];
                auto weights = [&](int pack, float (&w)[VEC]) {
                    if constexpr (VEC % 4 == 0) {
#pragma unroll
                        for (int j = 0; j < VEC; j += 4) {
                            const float4 v = *reinterpret_cast<const float4*>(&s_w[kind][max(pack, 0) * VEC + j]);
                            w[j] = v.x, w[j + 1] = v.y, w[j + 2] = v.z, w[j + 3] = v.w;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) w[j] = s_w[kind][max(pack, 0) * VEC + j];
                    }
                };
                for (int n = 0; n < turnsOf; ++n) {
                    Row y;
                    if (n + 1 < turnsOf) next(y);
                    float a[NI][VEC], b[NI][VEC];
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        x.a[i].get(a[i]);
                        x.b[i].get(b[i]);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            if (!x.out || ia[i] < 0) a[i][j] = 0.f;
                            if (!x.out || ib[i] < 0) b[i][j] = 0.f;
                            ss = fmaf(a[i][j], a[i][j], ss);
                            ss = fmaf(b[i][j], b[i][j], ss);
                        }
                    }
                    const float2* turn = s_turn + x.tt * pairs;
                    if constexpr (MODE != kGradient) {
                        float r = 1.f;
                        if (normed) {
                            for (int o = p.lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
                            r = __frsqrt_rn(ss * inv_dim + p.eps[kind]);
                        }
                        if (x.out) {
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                float wa[VEC], wb[VEC];
                                weights(ia[i], wa);
                                weights(ib[i], wb);
#pragma unroll
                                for (int j = 0; j < VEC; ++j) {
                                    a[i][j] = a[i][j] * r * wa[j];
                                    b[i][j] = b[i][j] * r * wb[j];
                                }
                            }
                            rotate(a, b, turn);
                        }
                    } else {
                        float ga[NI][VEC], gb[NI][VEC];
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            x.ga[i].get(ga[i]);
                            x.gb[i].get(gb[i]);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) {
                                if (!x.out || ia[i] < 0) ga[i][j] = 0.f;
                                if (!x.out || ib[i] < 0) gb[i][j] = 0.f;
                            }
                        }
                        if (x.out) rotate(ga, gb, turn);
                        if (normed) {
                            float dot = 0.f;
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                float wa[VEC], wb[VEC];
                                weights(ia[i], wa);
                                weights(ib[i], wb);
#pragma unroll
                                for (int j = 0; j < VEC; ++j) {
                                    dot = fmaf(ga[i][j] * wa[j], a[i][j], dot);
                                    dot = fmaf(gb[i][j] * wb[j], b[i][j], dot);
                                }
                            }
                            for (int o = p.lanes >> 1; o; o >>= 1) {
                                ss += __shfl_xor_sync(kFull, ss, o);
                                dot += __shfl_xor_sync(kFull, dot, o);
                            }
                            // eps = 0 and a row of zeros: r is infinite; rows of none leave acc alone
                            const float r = x.out ? __frsqrt_rn(ss * inv_dim + p.eps[kind]) : 0.f;
                            const float m = dot * r * inv_dim;
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                float wa[VEC], wb[VEC];
                                weights(ia[i], wa);
                                weights(ib[i], wb);
#pragma unroll
                                for (int j = 0; j < VEC; ++j) {
                                    const float xa = a[i][j] * r, xb = b[i][j] * r;
                                    a[i][j] = r * (ga[i][j] * wa[j] - xa * m);
                                    b[i][j] = r * (gb[i][j] * wb[j] - xb * m);
                                    acc[kind][i][0][j] = fmaf(ga[i][j], xa, acc[kind][i][0][j]);
                                    acc[kind][i][1][j] = fmaf(gb[i][j], xb, acc[kind][i][1][j]);
                                }
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < NI; ++i)
#pragma unroll
                                for (int j = 0; j < VEC; ++j) a[i][j] = ga[i][j], b[i][j] = gb[i][j];
                        }
                    }
                    if (x.out) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            x.a[i].put(a[i]);
                            x.b[i].put(b[i]);
                        }
                        store(x);
                    }
                    x = y;
                }
            }
        };
        rows_of(std::integral_constant<int, 0>());
        rows_of(std::integral_constant<int, 1>());
        if constexpr (kKinds == 3) rows_of(std::integral_constant<int, 2>());
    }

    if constexpr (MODE == kGradient) {
        // the groups of a warp, then the warps one after the other
        float* const s_sum = reinterpret_cast<float*>(s_turn4);  // [warp][dim]
        constexpr int kWarps = kRopeThreads / 32;
        const int warp = tid >> 5;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int side = 0; side < 2; ++side)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float v = acc[k][i][side][j];
                        for (int o = 16; o >= p.lanes; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
                        const int at = side ? ib[i] : ia[i];
                        if ((tid & 31) < p.lanes && at >= 0) s_sum[warp * p.dim + at * VEC + j] = v;
                    }
            __syncthreads();
            for (int i = tid; i < p.dim; i += kRopeThreads) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v += s_sum[w * p.dim + i];
                p.part[((int64_t)blockIdx.x * 2 + k) * p.dim + i] = v;
            }
        }
    }
}

constexpr int kSumCols = 32, kSumRows = 8;

// dweight of a kind (blockIdx.y): the CTAs' sums, eight interleaved runs of them first.
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
#pragma unroll 4
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

// CTAs of the gradient: two on each SM at most (its registers), each the same number of rounds or one less.
int gradient_ctas(int64_t rounds) { return (int)std::min<int64_t>(rounds, 2 * kSMs); }

// Tokens of a round: enough that each group of lanes has a few rows for its share of the sines, but at
// least eight CTAs an SM (a few tokens are one CTA each).
int tile_of(int64_t tokens, int rows, int groups, int pairs) {
    int64_t tile = ceil_div(4ll * groups, std::max(rows, 1));
    tile = std::min<int64_t>({tile, kRopeTile, std::max<int64_t>(1, tokens / (kSMs * 8)),
                              pairs ? std::max<int64_t>(1, kRopeSmem / (pairs * 8)) : kRopeTile});
    return (int)tile;
}

template <typename T>
struct Shape {
    int vec, chunks, lanes, groups, tile;
    size_t smem;
};

// How rows are moved: by the or of all addresses and strides in bytes.
template <typename T>
Shape<T> shape_of(uint64_t all, int dim, int rot, bool half, int64_t tokens, int rows) {
    Shape<T> s;
    for (s.vec = 16 / (int)sizeof(T); s.vec > 1; s.vec = s.vec * (int)sizeof(T) == 16 ? s.vec / 2 : 1)
        if (all % (s.vec * sizeof(T)) == 0 && dim % s.vec == 0 && rot % (half ? 2 * s.vec : s.vec) == 0) break;
    s.chunks = half || s.vec == 1 ? rot / 2 / s.vec + ((dim - rot) / s.vec + 1) / 2 : (dim / s.vec + 1) / 2;
    const int items = s.vec >= 4 ? 1 : 4 / s.vec;
    for (s.lanes = 1; s.lanes * items < s.chunks;) s.lanes *= 2;
    s.groups = kRopeThreads / s.lanes;
    s.tile = tile_of(tokens, rows, s.groups, rot / 2);
    s.smem = (size_t)s.tile * (rot / 2) * sizeof(float2);
    return s;
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
    const Shape<T> s = shape_of<T>(all, p.dim, p.rot, half, p.tokens, rows);
    p.chunks = s.chunks, p.lanes = s.lanes, p.groups = s.groups, p.tile = s.tile;
    const int64_t rounds = ceil_div(p.tokens, p.tile);
    ctas = MODE == kGradient ? gradient_ctas(rounds) : (int)rounds;
    size_t smem = s.smem;
    if (MODE == kGradient) smem = std::max(smem, (size_t)(kRopeThreads / 32) * p.dim * sizeof(float));
    constexpr int WIDE = 16 / (int)sizeof(T);
    auto kernel = s.vec == WIDE       ? (half ? norm_rope_kernel<T, WIDE, true, MODE> : norm_rope_kernel<T, WIDE, false, MODE>)
                  : s.vec == WIDE / 2 ? (half ? norm_rope_kernel<T, WIDE / 2, true, MODE> : norm_rope_kernel<T, WIDE / 2, false, MODE>)
                                      : (half ? norm_rope_kernel<T, 1, true, MODE> : norm_rope_kernel<T, 1, false, MODE>);
    kernel<<<(unsigned)ctas, kRopeThreads, smem, st>>>(p);
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
            return set_error(TG_EINVAL, "%s: workspace of %zu bytes needed (got %zu)", op, need, workspace_bytes);
        if (reinterpret_cast<uintptr_t>(workspace) % 4) return set_error(TG_EINVAL, "%s: the workspace must be 4-byte aligned", op);
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
