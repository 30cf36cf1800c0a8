// The weighted sum of a routed row's expert outputs by its k weights, and its gradients, on
// gfx950: out[r] = sum_i w[r, i] y[slot(r, i)] in rank order, any number of experts.
#include "common.hpp"

namespace nsosx {

constexpr int kTopkMax = 16;
constexpr int kTopkMaxDim = 1 << 30;  // a lane's element, and the step behind the last, in int
constexpr int kZeroSlots = 4;  // of a wave that clears unused rows

template <int V, int DT>
__device__ __forceinline__ void row_load(const void* p, int64_t at, float (&v)[V]) {
    if constexpr (V == 8) load8<DT>(p, at, v);
    else v[0] = load_act<DT>(p, at);
}

template <int V, int DT>
__device__ __forceinline__ void row_store(void* p, int64_t at, const float (&v)[V]) {
    if constexpr (V == 8 && DT == NSOSX_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
        d[0] = make_float4(v[0], v[1], v[2], v[3]);
        d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) =
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
    } else {
        store_act<DT>(p, at, v[0]);
    }
}

// The row's slots and weights, the same in every lane; an entry past k, or whose slot no expert row
// has, gets weight 0 and slot -1.
template <int KT>
__device__ __forceinline__ void row_entries(const int32_t* __restrict__ slot_of,
                                            const float* __restrict__ weights, int64_t r, int k, int slots,
                                            int (&s)[KT], float (&w)[KT]) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        const int64_t at = r * k + (i < k ? i : 0);
        s[i] = slot_of[at];
        w[i] = weights[at];
    }
#pragma unroll
    for (int i = 0; i < KT; ++i)
        if (i >= k || s[i] < 0 || s[i] >= slots) {
            s[i] = -1;
            w[i] = 0.0f;
        }
}

// A wave per 64 V elements of a row, the loads of KT >= k expert rows in flight together.
template <int IDT, int ODT, int V, int KT>
__global__ __launch_bounds__(256) void combine_topk_kernel(const void* __restrict__ expert_out,
                                                           const int32_t* __restrict__ slot_of,
                                                           const float* __restrict__ weights,
                                                           int rows, int slots, int k, int dim,
                                                           int pieces, void* __restrict__ out) {
    const int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (task >= (int64_t)rows * pieces) return;
    const int64_t r = task / pieces;
    const int d = ((int)(task - r * pieces) * 64 + (threadIdx.x & 63)) * V;
    int s[KT];
    float w[KT];
    row_entries<KT>(slot_of, weights, r, k, slots, s, w);
    if (d >= dim) return;
    float v[KT][V], acc[V];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        if (s[i] >= 0) {
            row_load<V, IDT>(expert_out, (int64_t)s[i] * dim + d, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = __fmaf_rn(v[i][j], w[i], acc[j]);
    row_store<V, ODT>(out, r * dim + d, acc);
}

// A workgroup per row, of up to 4 waves: the waves take the row's pieces in turn, each holds its
// part of the k dot products, and the parts are added in wave order.  The workgroups behind the
// rows' (where perm is given) write zeros into the rows of dexpert that no row holds (perm < 0):
// as a launch of their own they took 4.6 us.  4096 rows of 8 x 2048 bf16: 50 us, 5.7 TB/s of the
// rows read and written, what a copy reaches.
template <int DDT, int EDT, int V, int KT>
__global__ __launch_bounds__(256) void combine_topk_bwd_kernel(const void* __restrict__ dout,
                                                               const void* __restrict__ expert_out,
                                                               const int32_t* __restrict__ slot_of,
                                                               const float* __restrict__ weights,
                                                               const int32_t* __restrict__ perm,
                                                               int rows, int slots, int k, int dim,
                                                               void* __restrict__ dexpert,
                                                               float* __restrict__ dweights) {
    __shared__ float s_dot[4][kTopkMax];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    if ((int)blockIdx.x >= rows) {
        // (a few slots a wave: the empty ones lie together, at the end)
        const int64_t s0 = ((int64_t)(blockIdx.x - rows) * waves + wave) * kZeroSlots;
        uint64_t empty = __ballot(lane < kZeroSlots && s0 + lane < slots &&
                                  perm[min(s0 + lane, (int64_t)slots - 1)] < 0);
        const float zero[V] = {};
        for (; empty; empty &= empty - 1) {
            const int64_t row = s0 + __builtin_ctzll(empty);
            for (int d = lane * V; d < dim; d += kWave * V) row_store<V, EDT>(dexpert, row * dim + d, zero);
        }
        return;
    }
    const int64_t r = blockIdx.x;
    if constexpr (V == 8) {
        // one expert row after the other: 16-byte loads of enough workgroups keep the memory busy (all
        // of them in flight together were 54 us where this takes 49)
        for (int i = 0; i < k; ++i) {
            const int s = slot_of[r * k + i];
            float dot = 0.0f;
            if (s >= 0 && s < slots) {
                const float w = weights[r * k + i];
                for (int d = (wave * 64 + lane) * V; d < dim; d += waves * 64 * V) {
                    float g[V], v[V];
                    row_load<V, DDT>(dout, r * dim + d, g);
                    row_load<V, EDT>(expert_out, (int64_t)s * dim + d, v);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        dot = __fmaf_rn(g[j], v[j], dot);
                        g[j] = g[j] * w;
                    }
                    row_store<V, EDT>(dexpert, (int64_t)s * dim + d, g);
                }
            }
            dot = wave_sum(dot);
            if (lane == 0) s_dot[wave][i] = dot;
        }
    } else {
        // a row that is no multiple of 8, or not aligned: many small loads, all choices' together
        int s[KT];
        float w[KT], dot[KT];
        row_entries<KT>(slot_of, weights, r, k, slots, s, w);
#pragma unroll
        for (int i = 0; i < KT; ++i) dot[i] = 0.0f;
        for (int d = wave * 64 + lane; d < dim; d += waves * 64) {
            float v[KT];
            const float g = load_act<DDT>(dout, r * dim + d);
#pragma unroll
            for (int i = 0; i < KT; ++i)
                v[i] = s[i] >= 0 ? load_act<EDT>(expert_out, (int64_t)s[i] * dim + d) : 0.0f;
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                if (s[i] < 0) continue;
                dot[i] = __fmaf_rn(g, v[i], dot[i]);
                store_act<EDT>(dexpert, (int64_t)s[i] * dim + d, g * w[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const float sum = wave_sum(dot[i]);
            if (lane == 0) s_dot[wave][i] = sum;
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < k) {
        float sum = s_dot[0][threadIdx.x];
        for (int w = 1; w < waves; ++w) sum += s_dot[w][threadIdx.x];
        dweights[r * k + threadIdx.x] = sum;
    }
}

static bool vector_rows(int dim, const void* a, const void* b, const void* c) {
    return dim % 8 == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
                             reinterpret_cast<uintptr_t>(c)) & 15) == 0;
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int nsosx_moe_combine_topk(const void* expert_out, int in_dtype, const int32_t* slot_of,
                                      const float* weights, int rows, int slots, int k, int dim,
                                      void* out, int out_dtype, void* stream) {
    if (!expert_out || !slot_of || !weights || !out)
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk: null pointer");
    if (rows <= 0 || slots <= 0 || k <= 0 || k > kTopkMax || dim <= 0)
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk: need positive sizes and k <= 16");
    if (!valid_dtype(in_dtype) || !valid_dtype(out_dtype))
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk: bad dtype");
    if (overlaps(out, (int64_t)rows * dim * (out_dtype == NSOSX_F32 ? 4 : 2), expert_out,
                 (int64_t)slots * dim * (in_dtype == NSOSX_F32 ? 4 : 2)))
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk: out overlaps expert_out");
    const bool v8 = vector_rows(dim, expert_out, out, nullptr);
    const int pieces = (dim - 1) / (v8 ? 512 : 64) + 1;
    const int64_t grid = ((int64_t)rows * pieces + 3) / 4;
    if (dim > kTopkMaxDim || grid > 0x7fffffffLL / 256)  // a launch holds less than 2^32 threads
        return fail(NSOSX_ERR_OVERFLOW, "moe_combine_topk: dim or rows * dim too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NSOSX_CT_K(I, O, V)                                                                        \
    do {                                                                                           \
        if (k <= 2) NSOSX_CT_L(I, O, V, 2);                                                        \
        else if (k <= 4) NSOSX_CT_L(I, O, V, 4);                                                   \
        else if (k <= 8) NSOSX_CT_L(I, O, V, 8);                                                   \
        else NSOSX_CT_L(I, O, V, 16);                                                              \
    } while (0)
#define NSOSX_CT_L(I, O, V, KT)                                                                    \
    hipLaunchKernelGGL((combine_topk_kernel<I, O, V, KT>), dim3((unsigned)grid), dim3(256), 0, st, \
                       expert_out, slot_of, weights, rows, slots, k, dim, pieces, out)
#define NSOSX_CT(I, O)                       \
    do {                                     \
        if (v8) NSOSX_CT_K(I, O, 8);         \
        else NSOSX_CT_K(I, O, 1);            \
    } while (0)
    if (in_dtype == NSOSX_F32) {
        if (out_dtype == NSOSX_F32) NSOSX_CT(NSOSX_F32, NSOSX_F32);
        else NSOSX_CT(NSOSX_F32, NSOSX_BF16);
    } else {
        if (out_dtype == NSOSX_F32) NSOSX_CT(NSOSX_BF16, NSOSX_F32);
        else NSOSX_CT(NSOSX_BF16, NSOSX_BF16);
    }
#undef NSOSX_CT_L
#undef NSOSX_CT_K
#undef NSOSX_CT
    return check_launch("moe_combine_topk");
}

extern "C" int nsosx_moe_combine_topk_backward(const void* dout, int dout_dtype,
                                               const void* expert_out, int expert_dtype,
                                               const int32_t* slot_of, const float* weights,
                                               const int32_t* perm, int rows, int slots, int k,
                                               int dim, void* dexpert, float* dweights,
                                               void* stream) {
    if (!dout || !expert_out || !slot_of || !weights || !dexpert || !dweights)
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk_backward: null pointer");
    if (rows <= 0 || slots <= 0 || k <= 0 || k > kTopkMax || dim <= 0)
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk_backward: need positive sizes and k <= 16");
    if (!valid_dtype(dout_dtype) || !valid_dtype(expert_dtype))
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk_backward: bad dtype");
    const int64_t db = (int64_t)rows * dim * (dout_dtype == NSOSX_F32 ? 4 : 2);
    const int64_t eb = (int64_t)slots * dim * (expert_dtype == NSOSX_F32 ? 4 : 2);
    const int64_t kb = (int64_t)rows * k * 4;
    if (overlaps(dexpert, eb, expert_out, eb) || overlaps(dexpert, eb, dout, db) ||
        overlaps(dexpert, eb, slot_of, kb) || overlaps(dexpert, eb, weights, kb) ||
        (perm && overlaps(dexpert, eb, perm, (int64_t)slots * 4)))
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk_backward: dexpert overlaps an input");
    if (overlaps(dexpert, eb, dweights, kb))
        return fail(NSOSX_ERR_INVALID, "moe_combine_topk_backward: dexpert overlaps dweights");
    const bool v8 = vector_rows(dim, dout, expert_out, dexpert);
    const int per = v8 ? 512 : 64;
    const int waves = dim > 2 * per ? 4 : dim > per ? 2 : 1;
    const int64_t grid = rows + (perm ? ((int64_t)slots - 1) / (kZeroSlots * waves) + 1 : 0);
    if (dim > kTopkMaxDim || grid > 0x7fffffffLL / 256)
        return fail(NSOSX_ERR_OVERFLOW, "moe_combine_topk_backward: rows, slots or dim too large");
    const dim3 block(64 * waves);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NSOSX_CB_L(D, E, V, KT)                                                                     \
    hipLaunchKernelGGL((combine_topk_bwd_kernel<D, E, V, KT>), dim3((unsigned)grid), block, 0, st, dout, \
                       expert_out, slot_of, weights, perm, rows, slots, k, dim, dexpert, dweights)
#define NSOSX_CB_K(D, E, V)                                                                         \
    do {                                                                                            \
        if (k <= 2) NSOSX_CB_L(D, E, V, 2);                                                         \
        else if (k <= 4) NSOSX_CB_L(D, E, V, 4);                                                    \
        else if (k <= 8) NSOSX_CB_L(D, E, V, 8);                                                    \
        else NSOSX_CB_L(D, E, V, 16);                                                               \
    } while (0)
#define NSOSX_CB(D, E)                       \
    do {                                     \
        if (v8) NSOSX_CB_L(D, E, 8, 16);     \
        else NSOSX_CB_K(D, E, 1);            \
    } while (0)
    if (dout_dtype == NSOSX_F32) {
        if (expert_dtype == NSOSX_F32) NSOSX_CB(NSOSX_F32, NSOSX_F32);
        else NSOSX_CB(NSOSX_F32, NSOSX_BF16);
    } else {
        if (expert_dtype == NSOSX_F32) NSOSX_CB(NSOSX_BF16, NSOSX_F32);
        else NSOSX_CB(NSOSX_BF16, NSOSX_BF16);
    }
#undef NSOSX_CB_L
#undef NSOSX_CB_K
#undef NSOSX_CB
    return check_launch("moe_combine_topk_backward");
}
