// Layer norm and its gradients on gfx950:
//   s = x (+ delta, as stored), mu = mean(s), v = mean((s - mu)^2), q = 1 / sqrt(v + eps)
//   y = (s - mu) q w + b
//   with n = (s - mu) q, g = dy w:  dx = q (g - mean(g) - n mean(g n)) (+ dresidual)
//   dw = sum_rows dy n,  db = sum_rows dy
// Every pass is bound by memory: a row is read once, held in registers (up to 16384 elements) by
// TPR threads of 8 CH elements each, and its sums are f32, the variance from the centred row.
#include "train.hpp"

namespace nsosx {

constexpr int kLnMaxDim = 1 << 30;
constexpr int kLnRegDim = 16384;  // longest row that is held in registers

// The sum over the TPR threads of a row, the same bits in each of them.  Rows of more than a wave add
// the waves' sums in wave order; `turn` alternates the LDS slots, so that one barrier is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* lds, int turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (TPR >= 64) v[i] += lane_xor<32>(v[i]);
        if constexpr (TPR >= 32) v[i] += lane_xor<16>(v[i]);
        if constexpr (TPR >= 16) v[i] += lane_xor<8>(v[i]);
        v[i] += lane_xor<4>(v[i]);
        v[i] += lane_xor<2>(v[i]);
        v[i] += lane_xor<1>(v[i]);
    }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int waves = blockDim.x >> 6;
        const int wave = threadIdx.x >> 6;
        float* at = lds + (turn & 1) * waves * N;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) at[wave * N + i] = v[i];
        }
        __syncthreads();
        const int first = wave / W * W;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = at[first * N + i];
#pragma unroll
            for (int w = 1; w < W; ++w) s += at[(first + w) * N + i];
            v[i] = s;
        }
    }
}

// y (and, with delta, the stored sum) of one row per TPR threads.
template <int DT, int ODT, int TPR, int CH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layernorm_kernel(
    const void* x, const void* delta, const float* __restrict__ weight,
    const float* __restrict__ bias, int rows, int dim, float eps, void* sum, void* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int NT = TPR > 256 ? TPR : 256;
    __shared__ float lds[2 * (NT / 64)];
    const int l = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
    const bool real = row < rows;
    const int64_t base = row * dim;
    float v[CH][8];
    int n[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        n[c] = real ? max(0, min(8, dim - (c * TPR + l) * 8)) : 0;
        load8_part<DT>(x, base + (c * TPR + l) * 8, n[c], v[c]);
    }
    if (delta) {
        float d[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) load8_part<DT>(delta, base + (c * TPR + l) * 8, n[c], d[c]);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = round_act<DT>(v[c][j] + d[c][j]);
            store8_part<DT>(sum, base + (c * TPR + l) * 8, n[c], v[c]);
        }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += v[c][j];
    row_sums<TPR, 1>(s, lds, 0);
    const float mean = s[0] / static_cast<float>(dim);
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[c][j] = c < CH - 1 || j < n[c] ? v[c][j] - mean : 0.0f;
            s[0] = __fmaf_rn(v[c][j], v[c][j], s[0]);
        }
    row_sums<TPR, 1>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(dim) + eps);
    if (real && l == 0 && mean_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * TPR + l) * 8;
        float w[8], b[8];
        if (weight) load8_part<NSOSX_F32>(weight, e, n[c], w);
        if (bias) load8_part<NSOSX_F32>(bias, e, n[c], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[c][j] *= rstd;
            if (weight && bias) v[c][j] = __fmaf_rn(v[c][j], w[j], b[j]);
            else if (weight) v[c][j] *= w[j];
            else if (bias) v[c][j] += b[j];
        }
        store8_part<ODT>(y, base + e, n[c], v[c]);
    }
}

// Rows past kLnRegDim: a workgroup of 1024 threads per row, which it reads again from the caches for
// the variance and for y.
template <int DT, int ODT>
__global__ __launch_bounds__(1024) void layernorm_long_kernel(
    const void* x, const void* delta, const float* __restrict__ weight,
    const float* __restrict__ bias, int dim, float eps, void* sum, void* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float lds[2 * 16];
    const int64_t base = (int64_t)blockIdx.x * dim;
    const void* src = delta ? sum : x;
    float s[1] = {0.0f};
    for (int e = threadIdx.x; e < dim; e += 1024) {
        float v = load_act<DT>(x, base + e);
        if (delta) {  // each thread reads again only what it stored itself
            v = round_act<DT>(v + load_act<DT>(delta, base + e));
            store_act<DT>(sum, base + e, v);
        }
        s[0] += v;
    }
    row_sums<1024, 1>(s, lds, 0);
    const float mean = s[0] / static_cast<float>(dim);
    s[0] = 0.0f;
    for (int e = threadIdx.x; e < dim; e += 1024) {
        const float d = load_act<DT>(src, base + e) - mean;
        s[0] = __fmaf_rn(d, d, s[0]);
    }
    row_sums<1024, 1>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(dim) + eps);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
    for (int e = threadIdx.x; e < dim; e += 1024) {
        float v = (load_act<DT>(src, base + e) - mean) * rstd;
        if (weight) v = __fmaf_rn(v, weight[e], bias ? bias[e] : 0.0f);
        else if (bias) v += bias[e];
        store_act<ODT>(y, base + e, v);
    }
}

// dx of a row per TPR threads, the rows in turn over the grid; each thread keeps its columns' sums of
// dy n and dy, which the workgroup adds in group order and leaves in part[0 / 1][workgroup][dim].
template <int DT, int GDT, int TPR, int CH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layernorm_bwd_kernel(
    const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ weight, const void* dres, int rows,
    int dim, void* dx, float* __restrict__ part) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    constexpr bool SHARE = GROUPS > 1;  // several rows a workgroup: their sums meet in LDS
    __shared__ float lds[2 * 2 * (NT / 64)];
    __shared__ float s_cols[SHARE ? 2 * TPR * 8 * CH : 1];
    const int l = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float w[CH][8], aw[CH][8], ab[CH][8];
    int n[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        n[c] = max(0, min(8, dim - (c * TPR + l) * 8));
        if (weight) load8_part<NSOSX_F32>(weight, (c * TPR + l) * 8, n[c], w[c]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!weight) w[c][j] = 1.0f;
            aw[c][j] = ab[c][j] = 0.0f;
        }
    }
    const float inv_dim = 1.0f / static_cast<float>(dim);
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < rows; r0 += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = r0 + group;
        const bool real = row < rows;
        const int64_t base = row * dim;
        float v[CH][8], g[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            load8_part<DT>(x, base + (c * TPR + l) * 8, real ? n[c] : 0, v[c]);
            load8_part<GDT>(dy, base + (c * TPR + l) * 8, real ? n[c] : 0, g[c]);
        }
        const float mu = real ? mean[row] : 0.0f, q = real ? rstd[row] : 0.0f;
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[c][j] = c < CH - 1 || j < n[c] ? (v[c][j] - mu) * q : 0.0f;
                aw[c][j] = __fmaf_rn(g[c][j], v[c][j], aw[c][j]);
                ab[c][j] += g[c][j];
                g[c][j] *= w[c][j];
                s[0] += g[c][j];
                s[1] = __fmaf_rn(g[c][j], v[c][j], s[1]);
            }
        row_sums<TPR, 2>(s, lds, turn++);
        const float m1 = s[0] * inv_dim, m2 = s[1] * inv_dim;
        if (!real) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[c][j] = q * (g[c][j] - m1 - v[c][j] * m2);
            if (dres) {
                float d[8];
                load8_part<DT>(dres, base + (c * TPR + l) * 8, n[c], d);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[c][j] += d[j];
            }
            store8_part<DT>(dx, base + (c * TPR + l) * 8, n[c], g[c]);
        }
    }
    if (!part) return;
    float* pw = part + (int64_t)blockIdx.x * dim;
    float* pb = pw + (int64_t)gridDim.x * dim;
    if constexpr (SHARE) {
        float* sw = s_cols;
        float* sb = s_cols + TPR * 8 * CH;
        for (int k = 0; k < GROUPS; ++k) {
            if (group == k) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int e = (c * TPR + l) * 8 + j;
                        sw[e] = k ? sw[e] + aw[c][j] : aw[c][j];
                        sb[e] = k ? sb[e] + ab[c][j] : ab[c][j];
                    }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < dim; e += NT) {
            pw[e] = sw[e];
            pb[e] = sb[e];
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            store8_part<NSOSX_F32>(pw, (c * TPR + l) * 8, n[c], aw[c]);
            store8_part<NSOSX_F32>(pb, (c * TPR + l) * 8, n[c], ab[c]);
        }
    }
}

// Rows past kLnRegDim: dx with a workgroup per row, in two readings of it.
template <int DT, int GDT>
__global__ __launch_bounds__(1024) void layernorm_bwd_long_kernel(
    const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ weight, const void* dres, int dim,
    void* dx) {
    __shared__ float lds[2 * 2 * 16];
    const int64_t base = (int64_t)blockIdx.x * dim;
    const float mu = mean[blockIdx.x], q = rstd[blockIdx.x];
    float s[2] = {0.0f, 0.0f};
    for (int e = threadIdx.x; e < dim; e += 1024) {
        const float n = (load_act<DT>(x, base + e) - mu) * q;
        const float g = load_act<GDT>(dy, base + e) * (weight ? weight[e] : 1.0f);
        s[0] += g;
        s[1] = __fmaf_rn(g, n, s[1]);
    }
    row_sums<1024, 2>(s, lds, 0);
    const float inv_dim = 1.0f / static_cast<float>(dim);
    const float m1 = s[0] * inv_dim, m2 = s[1] * inv_dim;
    for (int e = threadIdx.x; e < dim; e += 1024) {
        const float n = (load_act<DT>(x, base + e) - mu) * q;
        const float g = load_act<GDT>(dy, base + e) * (weight ? weight[e] : 1.0f);
        float d = q * (g - m1 - n * m2);
        if (dres) d += load_act<DT>(dres, base + e);
        store_act<DT>(dx, base + e, d);
    }
}

// ... and the columns' sums: a thread per column and run of rows.
template <int DT, int GDT>
__global__ __launch_bounds__(256) void layernorm_cols_kernel(
    const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, int rows, int dim, float* __restrict__ part) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= dim) return;
    float aw = 0.0f, ab = 0.0f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = load_act<GDT>(dy, r * dim + e);
        aw = __fmaf_rn(g, (load_act<DT>(x, r * dim + e) - mean[r]) * rstd[r], aw);
        ab += g;
    }
    part[(int64_t)blockIdx.y * dim + e] = aw;
    part[((int64_t)gridDim.y + blockIdx.y) * dim + e] = ab;
}

// 64 columns a workgroup; its 16 waves take every 16th partial row each, and meet in wave order.
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* __restrict__ part, int n,
                                                           int cols, float* out0, float* out1) {
    float* out = blockIdx.y ? out1 : out0;
    if (!out) return;
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const float* p = part + (int64_t)blockIdx.y * n * cols;
    float sum = 0.0f;
    if (c < cols)
        for (int r = wave; r < n; r += 16) sum += p[(int64_t)r * cols + c];
    s[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < cols) {
        for (int w = 1; w < 16; ++w) sum += s[w][lane];
        out[c] = sum;
    }
}

void launch_column_sums(const float* part, int arrays, int n, int cols, float* out0, float* out1,
                        hipStream_t st) {
    hipLaunchKernelGGL(column_sums_kernel, dim3((cols + 63) / 64, arrays), dim3(1024), 0, st, part,
                       n, cols, out0, out1);
}

// Threads a row and elements a thread (8 CH): as few threads as hold the row in registers.
struct LnShape { int tpr, ch; };

static LnShape ln_shape(int dim) {
    if (dim <= 64) return {8, 1};
    if (dim <= 128) return {16, 1};
    if (dim <= 256) return {32, 1};
    if (dim <= 2048) return {64, (dim + 511) / 512};
    if (dim <= 8192) return {256, (dim + 2047) / 2048};
    return {1024, 2};
}

#define NSOSX_LN_SHAPES(GO)                                                                     \
    switch (sh.tpr * 8 + sh.ch) {                                                               \
        case 8 * 8 + 1: GO(8, 1); break;                                                        \
        case 16 * 8 + 1: GO(16, 1); break;                                                      \
        case 32 * 8 + 1: GO(32, 1); break;                                                      \
        case 64 * 8 + 1: GO(64, 1); break;                                                      \
        case 64 * 8 + 2: GO(64, 2); break;                                                      \
        case 64 * 8 + 3: GO(64, 3); break;                                                      \
        case 64 * 8 + 4: GO(64, 4); break;                                                      \
        case 256 * 8 + 2: GO(256, 2); break;                                                    \
        case 256 * 8 + 3: GO(256, 3); break;                                                    \
        case 256 * 8 + 4: GO(256, 4); break;                                                    \
        default: GO(1024, 2); break;                                                            \
    }

// threads of the pass that gives a row to TPR threads (all but the gradients' short rows)
static int64_t ln_threads(int rows, int dim) {
    return (int64_t)rows * (dim > kLnRegDim ? 1024 : ln_shape(dim).tpr) + 1024;
}

constexpr int kLnWorkgroups = 512;  // of the backward pass at most: each leaves a row of partial sums

static int ln_bwd_workgroups(int rows, int dim) {
    if (dim > kLnRegDim) return rows < 64 ? rows : 64;
    const int tpr = ln_shape(dim).tpr, groups = tpr > 256 ? 1 : 256 / tpr;
    const int need = (rows + groups - 1) / groups;
    return need < kLnWorkgroups ? need : kLnWorkgroups;
}

template <int DT, int ODT>
static void launch_layernorm(const void* x, const void* delta, const float* weight,
                             const float* bias, int rows, int dim, float eps, void* sum, void* y,
                             float* mean, float* rstd, hipStream_t st) {
    if (dim > kLnRegDim) {
        hipLaunchKernelGGL((layernorm_long_kernel<DT, ODT>), dim3(rows), dim3(1024), 0, st, x, delta,
                           weight, bias, dim, eps, sum, y, mean, rstd);
        return;
    }
    const LnShape sh = ln_shape(dim);
    const int nt = sh.tpr > 256 ? sh.tpr : 256, groups = nt / sh.tpr;
    const dim3 grid((rows + groups - 1) / groups), block(nt);
#define NSOSX_LN(T, C)                                                                             \
    hipLaunchKernelGGL((layernorm_kernel<DT, ODT, T, C>), grid, block, 0, st, x, delta, weight, bias, \
                       rows, dim, eps, sum, y, mean, rstd)
    NSOSX_LN_SHAPES(NSOSX_LN)
#undef NSOSX_LN
}

template <int DT, int GDT>
static void launch_layernorm_bwd(const void* dy, const void* x, const float* mean, const float* rstd,
                                 const float* weight, const void* dres, int rows, int dim, void* dx,
                                 float* part, hipStream_t st) {
    const int wgs = ln_bwd_workgroups(rows, dim);
    if (dim > kLnRegDim) {
        hipLaunchKernelGGL((layernorm_bwd_long_kernel<DT, GDT>), dim3(rows), dim3(1024), 0, st, dy, x,
                           mean, rstd, weight, dres, dim, dx);
        if (part)
            hipLaunchKernelGGL((layernorm_cols_kernel<DT, GDT>), dim3((dim - 1) / 256 + 1, wgs),
                               dim3(256), 0, st, dy, x, mean, rstd, rows, dim, part);
        return;
    }
    const LnShape sh = ln_shape(dim);
    const dim3 grid(wgs), block(sh.tpr > 256 ? sh.tpr : 256);
#define NSOSX_LN(T, C)                                                                             \
    hipLaunchKernelGGL((layernorm_bwd_kernel<DT, GDT, T, C>), grid, block, 0, st, dy, x, mean, rstd, \
                       weight, dres, rows, dim, dx, part)
    NSOSX_LN_SHAPES(NSOSX_LN)
#undef NSOSX_LN
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int nsosx_layernorm(const void* x, const void* delta, const float* weight,
                               const float* bias, int rows, int dim, float eps, int act_dtype,
                               void* sum_out, void* y, int out_dtype, float* mean, float* rstd,
                               void* stream) {
    if (rows < 0 || dim <= 0) return fail(NSOSX_ERR_INVALID, "layernorm: need rows >= 0 and dim > 0");
    if (!valid_dtype(act_dtype) || !valid_dtype(out_dtype))
        return fail(NSOSX_ERR_INVALID, "layernorm: bad dtype");
    if (!(eps >= 0.0f) || eps > 3.0e38f) return fail(NSOSX_ERR_INVALID, "layernorm: eps must be finite and >= 0");
    if (rows == 0) return NSOSX_OK;
    if (!x || !y) return fail(NSOSX_ERR_INVALID, "layernorm: null pointer");
    if ((delta == nullptr) != (sum_out == nullptr))
        return fail(NSOSX_ERR_INVALID, "layernorm: delta and sum_out go together");
    if ((mean == nullptr) != (rstd == nullptr))
        return fail(NSOSX_ERR_INVALID, "layernorm: mean and rstd go together");
    const int64_t n = (int64_t)rows * dim, ib = n * dtype_bytes(act_dtype), ob = n * dtype_bytes(out_dtype);
    if (overlaps(y, ob, x, ib) || (delta && (overlaps(y, ob, delta, ib) || overlaps(y, ob, sum_out, ib))))
        return fail(NSOSX_ERR_INVALID, "layernorm: y overlaps an input or the sum");
    if (delta && (crosses(sum_out, ib, x, ib) || crosses(sum_out, ib, delta, ib)))
        return fail(NSOSX_ERR_INVALID, "layernorm: sum_out may be x or delta, but not cross them");
    if (dim > kLnMaxDim || ln_threads(rows, dim) > 0xffffffffLL)  // a launch holds less than 2^32 threads
        return fail(NSOSX_ERR_OVERFLOW, "layernorm: rows or dim too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NSOSX_LN_GO(I, O) \
    launch_layernorm<I, O>(x, delta, weight, bias, rows, dim, eps, sum_out, y, mean, rstd, st)
    if (act_dtype == NSOSX_F32) {
        if (out_dtype == NSOSX_F32) NSOSX_LN_GO(NSOSX_F32, NSOSX_F32);
        else NSOSX_LN_GO(NSOSX_F32, NSOSX_BF16);
    } else {
        if (out_dtype == NSOSX_F32) NSOSX_LN_GO(NSOSX_BF16, NSOSX_F32);
        else NSOSX_LN_GO(NSOSX_BF16, NSOSX_BF16);
    }
#undef NSOSX_LN_GO
    return check_launch("layernorm");
}

extern "C" int64_t nsosx_layernorm_backward_workspace(int rows, int dim) {
    if (rows < 0 || dim <= 0 || dim > kLnMaxDim) return 0;
    return (int64_t)2 * ln_bwd_workgroups(rows, dim) * dim * 4;
}

extern "C" int nsosx_layernorm_backward(const void* dy, int dy_dtype, const void* x,
                                        const float* mean, const float* rstd, const float* weight,
                                        const void* dresidual, int rows, int dim, int act_dtype,
                                        void* dx, float* dweight, float* dbias, void* workspace,
                                        void* stream) {
    if (rows < 0 || dim <= 0)
        return fail(NSOSX_ERR_INVALID, "layernorm_backward: need rows >= 0 and dim > 0");
    if (!valid_dtype(act_dtype) || !valid_dtype(dy_dtype))
        return fail(NSOSX_ERR_INVALID, "layernorm_backward: bad dtype");
    const bool cols = dweight || dbias;
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx || (cols && !workspace)))
        return fail(NSOSX_ERR_INVALID, "layernorm_backward: null pointer");
    const int64_t n = (int64_t)rows * dim, ib = n * dtype_bytes(act_dtype), gb = n * dtype_bytes(dy_dtype);
    if (rows > 0 && (overlaps(dx, ib, dy, gb) || overlaps(dx, ib, x, ib) ||
                     (dresidual && crosses(dx, ib, dresidual, ib))))
        return fail(NSOSX_ERR_INVALID, "layernorm_backward: dx overlaps an input (it may be dresidual)");
    if (dim > kLnMaxDim || ln_threads(rows, dim) > 0xffffffffLL)
        return fail(NSOSX_ERR_OVERFLOW, "layernorm_backward: rows or dim too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* part = cols ? static_cast<float*>(workspace) : nullptr;
#define NSOSX_LN_GO(I, G) \
    launch_layernorm_bwd<I, G>(dy, x, mean, rstd, weight, dresidual, rows, dim, dx, part, st)
    if (rows > 0) {
        if (act_dtype == NSOSX_F32) {
            if (dy_dtype == NSOSX_F32) NSOSX_LN_GO(NSOSX_F32, NSOSX_F32);
            else NSOSX_LN_GO(NSOSX_F32, NSOSX_BF16);
        } else {
            if (dy_dtype == NSOSX_F32) NSOSX_LN_GO(NSOSX_BF16, NSOSX_F32);
            else NSOSX_LN_GO(NSOSX_BF16, NSOSX_BF16);
        }
    }
#undef NSOSX_LN_GO
    if (cols) launch_column_sums(part, 2, ln_bwd_workgroups(rows, dim), dim, dweight, dbias, st);
    return check_launch("layernorm_backward");
}
