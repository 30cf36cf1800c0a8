// Scored expert routing on gfx950: softmax or sigmoid scores, a balance bias that takes part in
// the choice only, expert groups, top-k, renormalised and scaled weights, the dispatch to
// expert segments, and the gradient of the logits from that of the weights.
#include "common.hpp"

namespace nsosx {

constexpr int kScoredMaxExperts = 512, kScoredMaxK = 16, kScoredMaxGroups = 16;

struct RouteScored {
    const void* logits;
    int64_t stride;          // elements between rows
    const uint8_t* valid;
    const float* bias;
    int rows, E, k;
    int sigmoid, groups, keep, best, renorm;
    float scale;
    float* weights;          // [rows, k]
    int32_t* selected;       // [rows, k]
    int32_t* counts;         // [E]; null: selection only
    int32_t* offsets;        // [E + 1]
    int32_t* perm;           // [rows * k]
    int32_t* slot_of;        // [rows, k]
    int32_t* block_counts;   // workspace [E, blocks]
};

// ---- sixteen lanes per row -----------------------------------------------------
// A row's experts lie on the 16 lanes of a DPP row, expert 16 v + l in value v of lane l, so
// that four rows share a wave and every reduction over a row is four rotations.

template <int N>
__device__ __forceinline__ uint32_t ror16(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x120 + N, 0xF, 0xF, true);
}
template <int N>
__device__ __forceinline__ int ror16(int v) { return (int)ror16<N>((uint32_t)v); }
template <int N>
__device__ __forceinline__ float ror16(float v) {
    return __uint_as_float(ror16<N>(__float_as_uint(v)));
}
template <int N>
__device__ __forceinline__ double ror16(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = ror16<N>((uint32_t)u), hi = ror16<N>((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, lo | (hi << 32));
}

template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }

template <typename T>
__device__ __forceinline__ T row_max(T v) {
    v = larger(v, ror16<8>(v));
    v = larger(v, ror16<4>(v));
    v = larger(v, ror16<2>(v));
    return larger(v, ror16<1>(v));
}
template <typename T>
__device__ __forceinline__ T row_sum(T v) {
    v = v + ror16<8>(v);
    v = v + ror16<4>(v);
    v = v + ror16<2>(v);
    return v + ror16<1>(v);
}
__device__ __forceinline__ bool row_any(bool p) {
    return ((__ballot(p) >> (threadIdx.x & 48)) & 0xFFFF) != 0;
}

// The two largest of a row from each lane's two largest (a >= b).
template <typename T, int N>
__device__ __forceinline__ void merge2(T& a, T& b) {
    const T oa = ror16<N>(a), ob = ror16<N>(b);
    b = larger(a < oa ? a : oa, larger(b, ob));
    a = larger(a, oa);
}

// Score of group `q` (its best one or two values in c; unavailable experts, -inf, add nothing),
// the same in every lane of the row; -inf where no expert of it is available.
template <typename T, int V>
__device__ __forceinline__ T group_score(const T (&c)[V], int q, int size, int best) {
    const T none = -(T)INFINITY;
    const int l = threadIdx.x & 15;
    T a = none, b = none;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (16 * v + 15 < q * size || 16 * v >= (q + 1) * size) continue;
        const int e = 16 * v + l;
        const T x = e >= q * size && e < (q + 1) * size ? c[v] : none;
        b = larger(b, a < x ? a : x);
        a = larger(a, x);
    }
    merge2<T, 8>(a, b);
    merge2<T, 4>(a, b);
    merge2<T, 2>(a, b);
    merge2<T, 1>(a, b);
    return best == 2 && b > none ? a + b : a;
}

template <int N, typename T>
__device__ __forceinline__ void outranked(T s, int l, int& rank) {
    const T o = ror16<N>(s);
    const int ol = ror16<N>(l);
    rank += o > s || (o == s && ol < l) ? 1 : 0;
}

// Bit q of the result: group q is one of the `keep` best (ties to the lower group).
template <typename T, int V>
__device__ __forceinline__ uint32_t kept_groups(const T (&c)[V], const RouteScored& p) {
    const int l = threadIdx.x & 15;
    const int size = p.E / p.groups;
    T s = -(T)INFINITY;
    for (int q = 0; q < p.groups; ++q) {
        const T v = group_score<T, V>(c, q, size, p.best);
        if (l == q) s = v;
    }
    int rank = 0;
    outranked<1>(s, l, rank); outranked<2>(s, l, rank); outranked<3>(s, l, rank);
    outranked<4>(s, l, rank); outranked<5>(s, l, rank); outranked<6>(s, l, rank);
    outranked<7>(s, l, rank); outranked<8>(s, l, rank); outranked<9>(s, l, rank);
    outranked<10>(s, l, rank); outranked<11>(s, l, rank); outranked<12>(s, l, rank);
    outranked<13>(s, l, rank); outranked<14>(s, l, rank); outranked<15>(s, l, rank);
    const bool in = l < p.groups && rank < p.keep;
    return (uint32_t)(__ballot(in) >> (threadIdx.x & 48)) & 0xFFFFu;
}

// The scores' sum and maximum of a softmax row, in T (unavailable experts are -inf).
template <typename T, int V>
__device__ __forceinline__ void softmax_stats(const T (&x)[V], T& mx, T& sum) {
    mx = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) mx = larger(mx, x[v]);
    mx = row_max(mx);
    sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += x[v] == -(T)INFINITY ? (T)0 : exp(x[v] - mx);  // a NaN stays
    sum = row_sum(sum);
}

// The row's choice values in 64 bits, then k rounds of a row maximum: expert index of choice
// l in lane l (-1 where no expert is left).
template <int V, int DT>
__device__ __forceinline__ int select_row(const RouteScored& p, int64_t row, bool live, bool& bad) {
    const double none = -(double)INFINITY;
    const int l = threadIdx.x & 15;
    double c[V];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = 16 * v + l;
        c[v] = live && e < p.E ? (double)load_act<DT>(p.logits, row * p.stride + e) : none;
        nan |= c[v] != c[v];
    }
    if (p.sigmoid) {
        if (p.bias || (p.groups > 1 && p.best == 2)) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (c[v] > none) c[v] = 1.0 / (1.0 + exp(-c[v]));
        }
    } else {
        double mx, sum;
        softmax_stats<double, V>(c, mx, sum);
        nan |= mx == (double)INFINITY;
        if (p.bias || (p.groups > 1 && p.best == 2)) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (c[v] > none) c[v] = exp(c[v] - mx) / sum;
        }
    }
    if (p.bias) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = 16 * v + l;
            if (e < p.E && c[v] > none) c[v] += (double)p.bias[e];
            nan |= c[v] != c[v];
        }
    }
    bad = row_any(nan);
    if (p.groups > 1) {
        const uint32_t kept = kept_groups<double, V>(c, p);
        const int size = p.E / p.groups;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = 16 * v + l;
            if (e < p.E && !((kept >> (e / size)) & 1)) c[v] = none;
        }
    }
    int mine = -1;
    for (int i = 0; i < p.k; ++i) {
        double bv = none;
        int be = 0x7fffffff;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (c[v] > bv) {  // ties keep the lower index
                bv = c[v];
                be = 16 * v + l;
            }
#define NSOSX_STEP(N)                                                   \
    {                                                                   \
        const double ov = ror16<N>(bv);                                 \
        const int oe = ror16<N>(be);                                    \
        if (ov > bv || (ov == bv && oe < be)) { bv = ov; be = oe; }     \
    }
        NSOSX_STEP(8) NSOSX_STEP(4) NSOSX_STEP(2) NSOSX_STEP(1)
#undef NSOSX_STEP
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (be == 16 * v + l) c[v] = none;
        if (l == i) mine = bv > none ? be : -1;
    }
    return mine;
}

// Weight of choice l in lane l (0 where mine < 0).  Renormalised weights are a softmax over
// the chosen logits (softmax scores: the common denominator drops out) or the sigmoids over
// their sum, both with the common factor exp(min(max, 0)) taken out, so that no sum underflows.
template <int V, int DT>
__device__ __forceinline__ float row_weight(const RouteScored& p, int64_t row, bool live, int mine) {
    const int l = threadIdx.x & 15;
    const float none = -INFINITY;
    const float x = mine >= 0 ? load_act<DT>(p.logits, row * p.stride + mine) : none;
    float t;
    if (!p.renorm) {
        if (p.sigmoid) {
            t = x > 0.0f ? 1.0f / (1.0f + expf(-x)) : expf(x) / (1.0f + expf(x));
        } else {
            float all[V], mx, sum;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int e = 16 * v + l;
                all[v] = live && e < p.E ? load_act<DT>(p.logits, row * p.stride + e) : none;
            }
            softmax_stats<float, V>(all, mx, sum);
            t = expf(x - mx) / sum;
        }
        return mine >= 0 ? t * p.scale : 0.0f;
    }
    const float m = row_max(x);
    if (p.sigmoid)
        t = x > 0.0f ? 1.0f / (1.0f + expf(-x)) : expf(x - fminf(m, 0.0f)) / (1.0f + expf(x));
    else
        t = expf(x - m);
    t = mine >= 0 ? t : 0.0f;
    const float sum = row_sum(t);
    return mine >= 0 ? t / sum * p.scale : 0.0f;
}

// Exclusive scan of counts [E] into s_off [E + 1] by the first wave of a workgroup.
__device__ __forceinline__ void scan_counts(const int32_t* counts, int E, int32_t* s_off) {
    if (threadIdx.x >= kWave) return;
    const int lane = threadIdx.x;
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += kWave) {
        const int c = e0 + lane < E ? counts[e0 + lane] : 0;
        int upto = c;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int v = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += v;
        }
        if (e0 + lane < E) s_off[e0 + lane] = carry + upto - c;
        carry += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (lane == 0) s_off[E] = carry;
}

// A workgroup of 16 RB threads routes RB rows, ranks them per expert through 64-bit row masks
// and leaves its counts per expert, or, where it is the only one, the whole dispatch.
template <int V, int DT>
__global__ __launch_bounds__(V > 16 ? 512 : 1024) void route_scored_kernel(RouteScored p) {
    __shared__ uint64_t s_mask[kScoredMaxExperts];
    __shared__ int32_t s_cnt[kScoredMaxExperts], s_off[kScoredMaxExperts + 1];
    const int l = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int row = blockIdx.x * (blockDim.x >> 4) + rl;
    const bool dispatch = p.counts != nullptr;
    if (dispatch) {
        for (int e = threadIdx.x; e < p.E; e += blockDim.x) s_mask[e] = 0;
        __syncthreads();
    }
    const bool live = row < p.rows && (!p.valid || p.valid[row] != 0);
    bool bad;
    int mine = select_row<V, DT>(p, row, live, bad);
    if (live && bad) mine = l < p.k ? l : -1;  // a NaN score: the first k experts, weights NaN
    float w = row_weight<V, DT>(p, row, live, mine);
    if (live && bad) w = NAN;
    const bool entry = row < p.rows && l < p.k;
    const int64_t at = (int64_t)row * p.k + l;
    if (entry) {
        p.weights[at] = w;
        p.selected[at] = mine;
    }
    if (!dispatch) return;
    const bool slot = entry && mine >= 0;
    if (slot) atomicOr((unsigned long long*)&s_mask[mine], 1ull << rl);
    __syncthreads();
    const int rank = slot ? __popcll(s_mask[mine] & ((1ull << rl) - 1)) : -1;
    if (gridDim.x > 1) {
        if (entry) p.slot_of[at] = rank;  // the rank within the block, until the placement
        for (int e = threadIdx.x; e < p.E; e += blockDim.x)
            p.block_counts[(int64_t)e * gridDim.x + blockIdx.x] = __popcll(s_mask[e]);
        return;
    }
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.counts[e] = s_cnt[e] = __popcll(s_mask[e]);
    __syncthreads();
    scan_counts(s_cnt, p.E, s_off);
    __syncthreads();
    for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = s_off[e];
    if (entry) {
        const int s = slot ? s_off[mine] + rank : -1;
        p.slot_of[at] = s;
        if (slot) p.perm[s] = row;
    }
    const int total = s_off[p.E];
    for (int i = total + threadIdx.x; i < p.rows * p.k; i += blockDim.x) p.perm[i] = -1;
}

// Per expert (a wave each): the exclusive scan of its counts over the blocks, in place.
__global__ __launch_bounds__(256) void route_scored_scan_kernel(int32_t* __restrict__ block_counts,
                                                                int blocks, int E,
                                                                int32_t* __restrict__ counts) {
    const int e = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (e >= E) return;
    const int lane = threadIdx.x & 63;
    int32_t* row = block_counts + (int64_t)e * blocks;
    int carry = 0;
    for (int b0 = 0; b0 < blocks; b0 += kWave) {
        const int c = b0 + lane < blocks ? row[b0 + lane] : 0;
        int upto = c;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int v = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += v;
        }
        if (b0 + lane < blocks) row[b0 + lane] = carry + upto - c;
        carry += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (lane == 0) counts[e] = carry;
}

// Ranks within a block -> slots.
__global__ __launch_bounds__(256) void route_scored_place_kernel(RouteScored p, int blocks,
                                                                 int block_rows) {
    __shared__ int32_t s_off[kScoredMaxExperts + 1];
    scan_counts(p.counts, p.E, s_off);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= p.E; e += blockDim.x) p.offsets[e] = s_off[e];
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.rows * p.k) return;
    const int row = (int)(i / p.k), e = p.selected[i];
    if (e >= 0) {
        const int s = s_off[e] + p.block_counts[(int64_t)e * blocks + row / block_rows] + p.slot_of[i];
        p.slot_of[i] = s;
        p.perm[s] = row;
    }
    if (i >= s_off[p.E]) p.perm[i] = -1;
}

// ---- gradient ---------------------------------------------------------------------
// With w_i the weights and g_i their gradients times `scale` (chosen experts only):
//   renormalised, softmax scores   dx_i = w_i (g_i - sum_j g_j w_j)
//   renormalised, sigmoid scores   dx_i = w_i (g_i - sum_j g_j w_j) (1 - s_i)
//   sigmoid scores as they are     dx_i = g_i s_i (1 - s_i)
//   softmax scores as they are     dx_e = p_e (g_e - sum_j g_j p_j), for every expert
// (w here before the scale).  An expert named twice in a row gets both gradients.
struct RouteScoredBwd {
    const void* logits;
    int64_t stride;
    const int32_t* selected;
    const float* dweights;
    int rows, E, k;
    int sigmoid, renorm;
    float scale;
    void* dlogits;  // [rows, E], contiguous
};

template <int V, int DT>
__global__ __launch_bounds__(256) void route_scored_bwd_kernel(RouteScoredBwd p) {
    extern __shared__ float s_g[];  // [16, E]
    const int l = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int row = blockIdx.x * 16 + rl;
    const bool live = row < p.rows;
    for (int i = threadIdx.x; i < 16 * p.E; i += 256) s_g[i] = 0.0f;
    __syncthreads();
    const int64_t base = (int64_t)row * p.stride;
    const int64_t at = (int64_t)row * p.k + l;
    int e = live && l < p.k ? p.selected[at] : -1;
    if (e >= p.E) e = -1;
    const float none = -INFINITY;
    const float x = e >= 0 ? load_act<DT>(p.logits, base + e) : none;
    float g = e >= 0 ? p.dweights[at] * p.scale : 0.0f;
    const bool dense = !p.renorm && !p.sigmoid;
    float mx = none, sum = 1.0f, dot = 0.0f;
    float all[V];
    if (dense) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            all[v] = live && 16 * v + l < p.E ? load_act<DT>(p.logits, base + 16 * v + l) : none;
        softmax_stats<float, V>(all, mx, sum);
        dot = row_sum(e < 0 || x == none ? 0.0f : g * (expf(x - mx) / sum));
    } else if (p.renorm) {
        const float m = row_max(x);
        float t = p.sigmoid ? (x > 0.0f ? 1.0f / (1.0f + expf(-x))
                                        : expf(x - fminf(m, 0.0f)) / (1.0f + expf(x)))
                            : expf(x - m);
        t = e < 0 || x == none ? 0.0f : t;  // a NaN stays
        const float total = row_sum(t);
        const float w = total == 0.0f ? 0.0f : t / total;
        g = w * (g - row_sum(g * w));
        if (p.sigmoid) g = g * (1.0f / (1.0f + expf(x)));
    } else {
        const float s = x > 0.0f ? 1.0f / (1.0f + expf(-x)) : expf(x) / (1.0f + expf(x));
        g = g * s * (1.0f / (1.0f + expf(x)));
    }
    // one lane after the other, so that an expert named twice adds both
    for (int i = 0; i < p.k; ++i)
        if (l == i && e >= 0) s_g[rl * p.E + e] += g;
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int j = 16 * v + l;
        if (j >= p.E) continue;
        float d = s_g[rl * p.E + j];
        if (dense) d = all[v] == none ? 0.0f : (expf(all[v] - mx) / sum) * (d - dot);
        store_act<DT>(p.dlogits, (int64_t)row * p.E + j, d);
    }
}

static int scored_block_rows(int rows, int E) {
    if (rows <= 16) return 16;
    if (rows <= 32) return 32;
    const int most = E > 256 ? 32 : 64;
    if (rows <= 64) return most;
    return rows <= 4096 ? 16 : rows <= 8192 ? 32 : most;
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int64_t nsosx_moe_route_scored_workspace(int rows, int experts) {
    if (rows <= 0 || experts <= 0 || experts > kScoredMaxExperts) return 0;
    const int rb = scored_block_rows(rows, experts);
    return (int64_t)((rows - 1) / rb + 1) * experts;
}

#define NSOSX_SCORED_V(E, CALL)          \
    do {                                 \
        if ((E) <= 32) CALL(2);          \
        else if ((E) <= 64) CALL(4);     \
        else if ((E) <= 128) CALL(8);    \
        else if ((E) <= 256) CALL(16);   \
        else CALL(32);                   \
    } while (0)

extern "C" int nsosx_moe_route_scored(const void* logits, int logits_dtype, int64_t logits_stride,
                                      const uint8_t* valid_rows, const float* bias, int rows,
                                      int experts, int k, int sigmoid, int groups, int group_keep,
                                      int group_best, int renorm, float scale, float* weights,
                                      int32_t* selected, int32_t* counts, int32_t* offsets,
                                      int32_t* perm, int32_t* slot_of, int32_t* workspace,
                                      void* stream) {
    const bool select_only = !counts && !offsets && !perm && !slot_of && !workspace;
    if (!logits || !weights || !selected ||
        (!select_only && (!counts || !offsets || !perm || !slot_of || !workspace)))
        return fail(NSOSX_ERR_INVALID, "moe_route_scored: null pointer");
    if (!valid_dtype(logits_dtype)) return fail(NSOSX_ERR_INVALID, "moe_route_scored: bad dtype");
    if (rows <= 0 || experts <= 0 || experts > kScoredMaxExperts || k <= 0 || k > experts ||
        k > kScoredMaxK)
        return fail(NSOSX_ERR_INVALID,
                    "moe_route_scored: need rows > 0, 0 < k <= 16, k <= E <= 512");
    if (logits_stride < experts)
        return fail(NSOSX_ERR_INVALID, "moe_route_scored: logits_stride below E");
    if (groups <= 0 || groups > kScoredMaxGroups || experts % groups != 0 || group_keep <= 0 ||
        group_keep > groups || (group_best != 1 && group_best != 2))
        return fail(NSOSX_ERR_INVALID,
                    "moe_route_scored: need 1 .. 16 groups that divide E, 0 < group_keep <= groups, "
                    "group_best 1 or 2");
    if (k > group_keep * (experts / groups))
        return fail(NSOSX_ERR_INVALID, "moe_route_scored: k exceeds the experts of the kept groups");
    if ((int64_t)rows * k > 2147483647LL)
        return fail(NSOSX_ERR_OVERFLOW, "moe_route_scored: rows*k too large");
    const int rb = scored_block_rows(rows, experts);
    const int blocks = (rows - 1) / rb + 1;
    RouteScored p{logits, logits_stride, valid_rows, bias, rows, experts, k, sigmoid != 0,
                  group_keep == groups ? 1 : groups, group_keep, group_best, renorm != 0, scale,
                  weights, selected, counts, offsets, perm, slot_of, workspace};
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NSOSX_RS(V)                                                                             \
    do {                                                                                        \
        if (logits_dtype == NSOSX_F32)                                                          \
            hipLaunchKernelGGL((route_scored_kernel<V, NSOSX_F32>), dim3(blocks), dim3(16 * rb), \
                               0, st, p);                                                       \
        else                                                                                    \
            hipLaunchKernelGGL((route_scored_kernel<V, NSOSX_BF16>), dim3(blocks), dim3(16 * rb), \
                               0, st, p);                                                       \
    } while (0)
    NSOSX_SCORED_V(experts, NSOSX_RS);
#undef NSOSX_RS
    if (!select_only && blocks > 1) {
        hipLaunchKernelGGL(route_scored_scan_kernel, dim3((experts + 3) / 4), dim3(256), 0, st,
                           workspace, blocks, experts, counts);
        const int64_t entries = (int64_t)rows * k;
        hipLaunchKernelGGL(route_scored_place_kernel, dim3((unsigned)((entries + 255) / 256)),
                           dim3(256), 0, st, p, blocks, rb);
    }
    return check_launch("moe_route_scored");
}

extern "C" int nsosx_moe_route_scored_backward(const void* logits, int logits_dtype,
                                               int64_t logits_stride, const int32_t* selected,
                                               const float* dweights, int rows, int experts, int k,
                                               int sigmoid, int renorm, float scale, void* dlogits,
                                               void* stream) {
    if (!logits || !selected || !dweights || !dlogits)
        return fail(NSOSX_ERR_INVALID, "moe_route_scored_backward: null pointer");
    if (!valid_dtype(logits_dtype))
        return fail(NSOSX_ERR_INVALID, "moe_route_scored_backward: bad dtype");
    if (rows <= 0 || experts <= 0 || experts > kScoredMaxExperts || k <= 0 || k > experts ||
        k > kScoredMaxK)
        return fail(NSOSX_ERR_INVALID,
                    "moe_route_scored_backward: need rows > 0, 0 < k <= 16, k <= E <= 512");
    if (logits_stride < experts)
        return fail(NSOSX_ERR_INVALID, "moe_route_scored_backward: logits_stride below E");
    if ((int64_t)rows * k > 2147483647LL)
        return fail(NSOSX_ERR_OVERFLOW, "moe_route_scored_backward: rows*k too large");
    const RouteScoredBwd p{logits, logits_stride, selected, dweights, rows, experts, k, sigmoid != 0,
                           renorm != 0, scale, dlogits};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((rows - 1) / 16 + 1), block(256);
    const int smem = 16 * experts * 4;
#define NSOSX_RB(V)                                                                                  \
    do {                                                                                             \
        if (logits_dtype == NSOSX_F32)                                                               \
            hipLaunchKernelGGL((route_scored_bwd_kernel<V, NSOSX_F32>), grid, block, smem, st, p);   \
        else                                                                                         \
            hipLaunchKernelGGL((route_scored_bwd_kernel<V, NSOSX_BF16>), grid, block, smem, st, p);  \
    } while (0)
    NSOSX_SCORED_V(experts, NSOSX_RB);
#undef NSOSX_RB
    return check_launch("moe_route_scored_backward");
}
