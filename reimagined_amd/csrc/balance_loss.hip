// The router's balance loss, per-expert counts and its gradient on gfx950.  With p the
// normalised scores of a row (softmax, or sigmoids over their sum), N_s the valid rows of sequence
// s, M the sequences that have any, and count_se the choices of expert e in s:
//   loss = 1/M sum_s E sum_e (count_se / (k N_s)) (sum_r p_re / N_s)
//   dloss/dx_rj = E / (M k N_s^2) p_rj (count_sj - sum_e count_se p_re)  [(1 - sigmoid) for sigmoids]
// Sixteen lanes per row, as in the scored routing: the row's sums are four lane exchanges, the
// columns' sums stay in registers over a block of rows.
#include "train.hpp"

namespace nsosx {

constexpr int kBalRows = 128;   // of a block of the forward pass
constexpr int kBalMaxE = 512, kBalMaxK = 16;

struct Balance {
    const void* logits;
    int64_t stride;
    const int32_t* selected;
    const uint8_t* valid;
    const int32_t* cu;
    int S, rows, E, k;
};

__device__ __forceinline__ float sum16(float v) {
    v += lane_xor<8>(v);
    v += lane_xor<4>(v);
    v += lane_xor<2>(v);
    v += lane_xor<1>(v);
    return v;
}

__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, lane_xor<8>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<2>(v));
    return fmaxf(v, lane_xor<1>(v));
}

// The row's normalised scores, columns i * 16 + l; `rest`, for sigmoids, their 1 - sigmoid.
template <int DT, int NC, bool SIG, bool REST>
__device__ __forceinline__ void row_probs(const void* logits, int64_t base, int E, int l, float (&p)[NC],
                                          float (&rest)[NC]) {
    float mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = i * 16 + l;
        p[i] = c < E ? load_act<DT>(logits, base + c) : -INFINITY;
    }
    if constexpr (!SIG) {
#pragma unroll
        for (int i = 0; i < NC; ++i) mx = fmaxf(mx, p[i]);
        mx = max16(mx);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if constexpr (SIG) {
            const float e = expf(-fabsf(p[i])), big = 1.0f / (1.0f + e), small = e * big;
            if constexpr (REST) rest[i] = p[i] < 0.0f ? big : small;
            p[i] = p[i] < 0.0f ? small : big;
        } else {
            p[i] = i * 16 + l < E ? expf(p[i] - mx) : 0.0f;
        }
        sum += p[i];
    }
    const float inv = 1.0f / sum16(sum);
#pragma unroll
    for (int i = 0; i < NC; ++i) p[i] *= inv;
}

// One block of rows: for each sequence in it, the sums of p and the counts, left in slot block +
// sequence (no two pairs share one: along the rows each step raises one of them or both).
template <int DT, int NC, bool SIG>
__global__ __launch_bounds__(1024) void balance_sums_kernel(Balance P, float* __restrict__ part,
                                                            int32_t* __restrict__ counts,
                                                            int32_t* __restrict__ tokens) {
    __shared__ float s_sum[16][NC * 16];
    __shared__ int32_t s_count[NC * 16], s_tokens, s_first, s_last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = threadIdx.x & 15;
    const int64_t r0 = (int64_t)blockIdx.x * kBalRows, r1 = min(r0 + kBalRows, (int64_t)P.rows);
    int first = 0, last = 0;
    if (P.cu) {
        if (threadIdx.x == 0) s_first = P.S, s_last = -1;
        __syncthreads();
        for (int s = threadIdx.x; s < P.S; s += 1024)
            if (P.cu[s] < r1 && P.cu[s + 1] > r0 && P.cu[s] < P.cu[s + 1]) {
                atomicMin(&s_first, s);
                atomicMax(&s_last, s);
            }
        __syncthreads();
        first = s_first, last = s_last;
    }
    for (int s = first; s <= last; ++s) {
        const int64_t lo = P.cu ? max(r0, (int64_t)P.cu[s]) : r0, hi = P.cu ? min(r1, (int64_t)P.cu[s + 1]) : r1;
        if (lo >= hi) continue;
        for (int e = threadIdx.x; e < P.E; e += 1024) s_count[e] = 0;
        if (threadIdx.x == 0) s_tokens = 0;
        __syncthreads();
        float acc[NC];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) acc[i] = 0.0f;
        for (int64_t r = lo + (threadIdx.x >> 4); r < hi; r += 64) {
            if (P.valid && !P.valid[r]) continue;
            float p[NC], rest[NC];
            row_probs<DT, NC, SIG, false>(P.logits, r * P.stride, P.E, l, p, rest);
#pragma unroll
            for (int i = 0; i < NC; ++i) acc[i] += p[i];
            if (l < P.k) {
                const int e = P.selected[r * P.k + l];
                if (e >= 0 && e < P.E) atomicAdd(&s_count[e], 1);
            }
            ++mine;
        }
        if (l == 0 && mine) atomicAdd(&s_tokens, mine);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            acc[i] += lane_xor<16>(acc[i]);
            acc[i] += lane_xor<32>(acc[i]);
            if (lane < 16) s_sum[wave][i * 16 + l] = acc[i];
        }
        __syncthreads();
        const int64_t slot = (int64_t)blockIdx.x + s;
        for (int e = threadIdx.x; e < P.E; e += 1024) {
            float sum = s_sum[0][e];
            for (int w = 1; w < 16; ++w) sum += s_sum[w][e];
            part[slot * P.E + e] = sum;
            counts[slot * P.E + e] = s_count[e];
        }
        if (threadIdx.x == 0) tokens[slot] = s_tokens;
        __syncthreads();
    }
}

// A sequence: its blocks' sums in order.  512 threads a column pair of four runs of blocks.
__global__ __launch_bounds__(1024) void balance_finish_kernel(Balance P, const float* __restrict__ part,
                                                              const int32_t* __restrict__ pcounts,
                                                              const int32_t* __restrict__ ptokens,
                                                              int32_t* __restrict__ counts,
                                                              int32_t* __restrict__ tokens,
                                                              float* __restrict__ mean,
                                                              float* __restrict__ seq_loss) {
    __shared__ float s_sum[1024];
    __shared__ int32_t s_count[1024], s_tokens;
    __shared__ double s_loss[16];
    const int s = blockIdx.x;
    const int64_t lo = P.cu ? max(0, P.cu[s]) : 0, hi = P.cu ? min(P.rows, P.cu[s + 1]) : P.rows;
    const int64_t b0 = lo / kBalRows, b1 = hi > lo ? (hi - 1) / kBalRows + 1 : b0;
    const int cols = P.E <= 64 ? 64 : P.E <= 256 ? 256 : 512, runs = 1024 / cols;
    const int e = threadIdx.x % cols, run = threadIdx.x / cols;
    float sum = 0.0f;
    int32_t count = 0;
    if (threadIdx.x == 0) s_tokens = 0;
    __syncthreads();
    if (e < P.E)
        for (int64_t b = b0 + run; b < b1; b += runs) {
            sum += part[(b + s) * P.E + e];
            count += pcounts[(b + s) * P.E + e];
        }
    int32_t n = 0;
    for (int64_t b = b0 + threadIdx.x; b < b1; b += 1024) n += ptokens[b + s];
    if (n) atomicAdd(&s_tokens, n);
    s_sum[threadIdx.x] = sum;
    s_count[threadIdx.x] = count;
    __syncthreads();
    const int32_t total = s_tokens;
    double loss = 0.0;
    if (run == 0 && e < P.E) {
        for (int q = 1; q < runs; ++q) {
            sum += s_sum[q * cols + e];
            count += s_count[q * cols + e];
        }
        const float avg = total ? sum / static_cast<float>(total) : 0.0f;
        counts[(int64_t)s * P.E + e] = count;
        mean[(int64_t)s * P.E + e] = avg;
        loss = total ? (double)count * avg : 0.0;
    }
    for (int o = 32; o > 0; o >>= 1) loss += __shfl_xor(loss, o, 64);
    if ((threadIdx.x & 63) == 0) s_loss[threadIdx.x >> 6] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) loss += s_loss[w];
        tokens[s] = total;
        seq_loss[s] = total ? (float)(loss * P.E / ((double)P.k * total)) : 0.0f;
    }
}

// The mean over the sequences with a valid row.
__global__ __launch_bounds__(256) void balance_mean_kernel(const float* __restrict__ seq_loss,
                                                           const int32_t* __restrict__ tokens, int S,
                                                           float* __restrict__ loss) {
    __shared__ double s_sum[256];
    __shared__ int32_t s_some[256];
    double sum = 0.0;
    int32_t some = 0;
    for (int s = threadIdx.x; s < S; s += 256) {
        sum += seq_loss[s];
        some += tokens[s] > 0;
    }
    s_sum[threadIdx.x] = sum;
    s_some[threadIdx.x] = some;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 256; ++i) {
            sum += s_sum[i];
            some += s_some[i];
        }
        *loss = some ? (float)(sum / some) : 0.0f;
    }
}

template <int DT, int NC, bool SIG>
__global__ __launch_bounds__(256) void balance_bwd_kernel(Balance P, const int32_t* __restrict__ counts,
                                                          const int32_t* __restrict__ tokens, float scale,
                                                          const float* __restrict__ dloss, const void* add,
                                                          void* dlogits) {
    __shared__ int32_t s_seq[16], s_some;
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t r0 = (int64_t)blockIdx.x * 16;
    if (threadIdx.x < 16) s_seq[threadIdx.x] = P.cu ? -1 : 0;
    if (threadIdx.x == 0) s_some = 0;
    __syncthreads();
    int some = 0;
    for (int s = threadIdx.x; s < P.S; s += 256) {
        some += tokens[s] > 0;
        if (P.cu) {
            const int64_t lo = max((int64_t)P.cu[s], r0), hi = min((int64_t)P.cu[s + 1], r0 + 16);
            for (int64_t r = lo; r < hi; ++r) s_seq[r - r0] = s;
        }
    }
    if (some) atomicAdd(&s_some, some);
    __syncthreads();
    const int64_t r = r0 + group;
    if (r >= P.rows) return;
    const int s = s_seq[group];
    const int n = s >= 0 ? tokens[s] : 0;
    float g[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) g[i] = 0.0f;
    if (n > 0 && !(P.valid && !P.valid[r])) {
        float p[NC], rest[NC], dot = 0.0f;
        row_probs<DT, NC, SIG, true>(P.logits, r * P.stride, P.E, l, p, rest);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            g[i] = i * 16 + l < P.E ? static_cast<float>(counts[(int64_t)s * P.E + i * 16 + l]) : 0.0f;
            dot = __fmaf_rn(g[i], p[i], dot);
        }
        dot = sum16(dot);
        const float nf = static_cast<float>(n);
        const float f = scale * (dloss ? *dloss : 1.0f) * static_cast<float>(P.E) /
                        (static_cast<float>(P.k) * static_cast<float>(s_some) * nf) / nf;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            g[i] = p[i] * (g[i] - dot) * f;
            if constexpr (SIG) g[i] *= rest[i];
        }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = i * 16 + l;
        if (c >= P.E) continue;
        if (add) g[i] += load_act<DT>(add, r * P.E + c);
        store_act<DT>(dlogits, r * P.E + c, g[i]);
    }
}

static int64_t bal_blocks(int rows) { return ((int64_t)rows + kBalRows - 1) / kBalRows; }

#define NSOSX_BAL_NC(GO, DT, SIG)                 \
    do {                                          \
        if (p.E <= 16) GO(DT, 1, SIG);            \
        else if (p.E <= 32) GO(DT, 2, SIG);       \
        else if (p.E <= 64) GO(DT, 4, SIG);       \
        else if (p.E <= 128) GO(DT, 8, SIG);      \
        else if (p.E <= 256) GO(DT, 16, SIG);     \
        else GO(DT, 32, SIG);                     \
    } while (0)
#define NSOSX_BAL(GO, dtype, sig)                                                    \
    do {                                                                             \
        if ((dtype) == NSOSX_F32) {                                                  \
            if (sig) NSOSX_BAL_NC(GO, NSOSX_F32, true);                              \
            else NSOSX_BAL_NC(GO, NSOSX_F32, false);                                 \
        } else {                                                                     \
            if (sig) NSOSX_BAL_NC(GO, NSOSX_BF16, true);                             \
            else NSOSX_BAL_NC(GO, NSOSX_BF16, false);                                \
        }                                                                            \
    } while (0)

static int bal_check(const char* fn, const Balance& p, int dtype) {
    const std::string name(fn);
    if (p.rows < 0 || p.E <= 0 || p.E > kBalMaxE || p.k <= 0 || p.k > kBalMaxK || p.k > p.E)
        return fail(NSOSX_ERR_INVALID, name + ": need rows >= 0, 0 < E <= 512 and 0 < k <= 16, k <= E");
    if (!valid_dtype(dtype)) return fail(NSOSX_ERR_INVALID, name + ": bad dtype");
    if (p.S < 0 || (!p.cu && p.S != 1))
        return fail(NSOSX_ERR_INVALID, name + ": need sequences >= 0, 1 without cu_seqlens");
    if (p.rows > 1 && p.stride < p.E)
        return fail(NSOSX_ERR_INVALID, name + ": the logits' row stride is less than E");
    if ((int64_t)p.rows * 16 + 256 > 0xffffffffLL || p.S > 0xffffffffLL / 1024 - 1)
        return fail(NSOSX_ERR_OVERFLOW, name + ": rows or sequences too large");
    return NSOSX_OK;
}

}  // namespace nsosx

using namespace nsosx;

// workspace: per slot (block + sequence) E sums, E counts and the rows, then the sequences' losses
extern "C" int64_t nsosx_moe_balance_loss_workspace(int rows, int experts, int S) {
    if (rows < 0 || experts <= 0 || S < 0) return 0;
    return ((bal_blocks(rows) + S) * (2 * (int64_t)experts + 1) + S) * 4;
}

extern "C" int nsosx_moe_balance_loss(const void* logits, int logits_dtype, int64_t logits_stride,
                                      const int32_t* selected, const uint8_t* valid_rows, int rows,
                                      int experts, int k, int sigmoid, const int32_t* cu_seqlens, int S,
                                      float* loss, int32_t* counts, int32_t* tokens, float* mean_prob,
                                      void* workspace, void* stream) {
    const Balance p{logits, logits_stride, selected, valid_rows, cu_seqlens, S, rows, experts, k};
    if (const int rc = bal_check("moe_balance_loss", p, logits_dtype)) return rc;
    if (!loss || (S > 0 && (!counts || !tokens || !mean_prob || !workspace)) ||
        (rows > 0 && (!logits || !selected)))
        return fail(NSOSX_ERR_INVALID, "moe_balance_loss: null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = bal_blocks(rows), slots = blocks + S;
    float* part = static_cast<float*>(workspace);
    int32_t* pcounts = reinterpret_cast<int32_t*>(part + slots * experts);
    int32_t* ptokens = pcounts + slots * experts;
    float* seq_loss = reinterpret_cast<float*>(ptokens + slots);
#define NSOSX_BAL_GO(DT, NC, SIG)                                                                     \
    hipLaunchKernelGGL((balance_sums_kernel<DT, NC, SIG>), dim3((unsigned)blocks), dim3(1024), 0, st, p, \
                       part, pcounts, ptokens)
    if (rows > 0 && S > 0) NSOSX_BAL(NSOSX_BAL_GO, logits_dtype, sigmoid);
#undef NSOSX_BAL_GO
    if (S > 0)
        hipLaunchKernelGGL(balance_finish_kernel, dim3(S), dim3(1024), 0, st, p, part, pcounts, ptokens,
                           counts, tokens, mean_prob, S == 1 ? loss : seq_loss);
    if (S != 1)
        hipLaunchKernelGGL(balance_mean_kernel, dim3(1), dim3(256), 0, st, seq_loss, tokens, S, loss);
    return check_launch("moe_balance_loss");
}

extern "C" int nsosx_moe_balance_loss_backward(const void* logits, int logits_dtype,
                                               int64_t logits_stride, const int32_t* counts,
                                               const int32_t* tokens, const uint8_t* valid_rows, int rows,
                                               int experts, int k, int sigmoid, const int32_t* cu_seqlens,
                                               int S, float scale, const float* dloss, const void* add,
                                               void* dlogits, void* stream) {
    const Balance p{logits, logits_stride, nullptr, valid_rows, cu_seqlens, S, rows, experts, k};
    if (const int rc = bal_check("moe_balance_loss_backward", p, logits_dtype)) return rc;
    if (rows == 0) return NSOSX_OK;
    if (!logits || !dlogits || (S > 0 && (!counts || !tokens)))
        return fail(NSOSX_ERR_INVALID, "moe_balance_loss_backward: null pointer");
    const int64_t size = dtype_bytes(logits_dtype), out = (int64_t)rows * experts * size;
    if (overlaps(dlogits, out, logits, ((int64_t)(rows - 1) * logits_stride + experts) * size) ||
        (S > 0 && overlaps(dlogits, out, counts, (int64_t)S * experts * 4)) ||
        (add && crosses(dlogits, out, add, out)))
        return fail(NSOSX_ERR_INVALID, "moe_balance_loss_backward: dlogits overlaps an input (it may be add)");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(((int64_t)rows + 15) / 16));
#define NSOSX_BAL_GO(DT, NC, SIG)                                                                       \
    hipLaunchKernelGGL((balance_bwd_kernel<DT, NC, SIG>), grid, dim3(256), 0, st, p, counts, tokens, scale, \
                       dloss, add, dlogits)
    NSOSX_BAL(NSOSX_BAL_GO, logits_dtype, sigmoid);
#undef NSOSX_BAL_GO
    return check_launch("moe_balance_loss_backward");
}
