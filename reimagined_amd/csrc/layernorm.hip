// Layer norm and its gradients on gfx950:
//   s = x (+ delta, as stored), mu = mean(s), v = mean((s - mu)^2), q = 1 / sqrt(v + eps)
//   y = (s - mu) q w + b
//   with n = (s - mu) q, g = dy w:  dx = q (g - mean(g) - n mean(g n)) (+ dresidual)
//   dw = sum_rows dy n,  db = sum_rows dy
// Every pass is bound by memory: a row is read once, held in registers (up to 16384 elements) by
// TPR threads of 8 CH elements each, and its sums are f32, the variance from the centred row.
// 67 million bf16 places, add and norm (537 MB): 92 us at rows of 64 to 256 and of 1024 (5.8 TB/s), 94 to
// 100 at 2048 to 16384, 110 at 777, 121 at 32; the gradients with a residual (as much): 101 to 108 at
// 128 to 8192, 114 at 64, 181 at 16384.
#include "train.hpp"

namespace nsosx {

constexpr int kLnMaxDim = 1 << 30;
constexpr int kLnRegDim = 16384;  // longest row that is held in registers

// The sum over the TPR threads of a row, the same bits in each of them.  Rows of more than a wave add
// the waves' sums in wave order; `turn` alternates the LDS slots, so that one barrier is enough.  NT: of
// the workgroup.
template <int TPR, int N, int NT>
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
        constexpr int waves = NT / 64;
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

// Which of the workgroup's rows a thread works on: known to be one for a wave where a row takes whole waves,
// so that its addresses are a scalar and a lane's offset.
template <int TPR>
__device__ __forceinline__ int row_group() {
    const int g = threadIdx.x / TPR;
    return TPR >= 64 ? __builtin_amdgcn_readfirstlane(g) : g;
}

// A thread's eight elements of piece c of a row of dim >= 8.  Those that would pass the row's end are the
// last eight of it instead, `skip` of which are another thread's: they stay out of the sums and are
// computed and stored twice, the same.  So no row needs a path for its tail, whatever its length.
template <int TPR, int CH>
struct Elements {
    int at[CH], skip;  // skip: of the last piece; the others are whole
    __device__ __forceinline__ Elements(int l, int dim) {
#pragma unroll
        for (int c = 0; c < CH; ++c) at[c] = min((c * TPR + l) * 8, dim - 8);
        skip = min(((CH - 1) * TPR + l) * 8 - at[CH - 1], 8);
    }
    __device__ __forceinline__ bool mine(int c, int j) const { return c < CH - 1 || j >= skip; }
    __device__ __forceinline__ bool any(int c) const { return c < CH - 1 || skip < 8; }
};

// y (and, with delta, the stored sum) of one row per TPR threads.
template <int DT, int ODT, int TPR, int CH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layernorm_kernel(
    const void* x, const void* delta, const float* __restrict__ weight,
    const float* __restrict__ bias, int rows, int dim, float eps, void* sum, void* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int NT = TPR > 256 ? TPR : 256;
    __shared__ float lds[2 * (NT / 64)];
    const int l = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + row_group<TPR>();
    const bool real = row < rows;
    const int64_t base = (real ? row : rows - 1) * dim;
    const Elements<TPR, CH> el(l, dim);
    float v[CH][8];
    {
        Raw8<DT> r[CH], d[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) r[c].load(x, base + el.at[c]);
        if (delta) {
#pragma unroll
            for (int c = 0; c < CH; ++c) d[c].load(delta, base + el.at[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = delta ? round_act<DT>(r[c].get(j) + d[c].get(j)) : r[c].get(j);
        }
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += el.mine(c, j) ? v[c][j] : 0.0f;
    row_sums<TPR, 1, NT>(s, lds, 0);
    // (behind the sums: a sum over x or delta is read twice at a row's tail before it is written)
    if (delta && real) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (el.any(c)) store8_any<DT>(sum, base + el.at[c], v[c]);
    }
    const float mean = s[0] / static_cast<float>(dim);
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[c][j] -= mean;
            const float d = el.mine(c, j) ? v[c][j] : 0.0f;
            s[0] = __fmaf_rn(d, d, s[0]);
        }
    row_sums<TPR, 1, NT>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(dim) + eps);
    if (!real) return;
    if (l == 0 && mean_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float w[8], b[8];
        if (weight) load8_any<NSOSX_F32>(weight, el.at[c], w);
        if (bias) load8_any<NSOSX_F32>(bias, el.at[c], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[c][j] *= rstd;
            if (weight && bias) v[c][j] = __fmaf_rn(v[c][j], w[j], b[j]);
            else if (weight) v[c][j] *= w[j];
            else if (bias) v[c][j] += b[j];
        }
        if (el.any(c)) store8_any<ODT>(y, base + el.at[c], v[c]);
    }
}

// Rows past kLnRegDim (and below 8): a workgroup per row, which it reads again from the caches for the
// variance and for y.
template <int DT, int ODT, int NT>
__global__ __launch_bounds__(NT) void layernorm_long_kernel(
    const void* x, const void* delta, const float* __restrict__ weight,
    const float* __restrict__ bias, int dim, float eps, void* sum, void* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float lds[2 * (NT / 64)];
    const int64_t base = (int64_t)blockIdx.x * dim;
    const void* src = delta ? sum : x;
    float s[1] = {0.0f};
    for (int e = threadIdx.x; e < dim; e += NT) {
        float v = load_act<DT>(x, base + e);
        if (delta) {  // each thread reads again only what it stored itself
            v = round_act<DT>(v + load_act<DT>(delta, base + e));
            store_act<DT>(sum, base + e, v);
        }
        s[0] += v;
    }
    row_sums<NT, 1, NT>(s, lds, 0);
    const float mean = s[0] / static_cast<float>(dim);
    s[0] = 0.0f;
    for (int e = threadIdx.x; e < dim; e += NT) {
        const float d = load_act<DT>(src, base + e) - mean;
        s[0] = __fmaf_rn(d, d, s[0]);
    }
    row_sums<NT, 1, NT>(s, lds, 1);
    const float rstd = 1.0f / sqrtf(s[0] / static_cast<float>(dim) + eps);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
    for (int e = threadIdx.x; e < dim; e += NT) {
        float v = (load_act<DT>(src, base + e) - mean) * rstd;
        if (weight) v = __fmaf_rn(v, weight[e], bias ? bias[e] : 0.0f);
        else if (bias) v += bias[e];
        store_act<ODT>(y, base + e, v);
    }
}

// Threads of a workgroup of the gradients (a longer row takes 1024): eight waves share one row of partial
// sums.  16384 x 2048 bf16 with a residual: 8 elements a thread in 128 registers 49 us, 16 elements 54 - 58
// (they spill), workgroups of 256 51.  Rows past 8192 have no more threads to give and take 16 each; with the
// weights held too 4096 x 16384 took 215 us, without 181 (16 to 24 registers spilled), reading the rows twice 308.
constexpr int kLnBwdThreads = 512;

template <int TPR> constexpr int ln_bwd_threads() { return TPR > kLnBwdThreads ? TPR : kLnBwdThreads; }

// dx of a row per TPR threads, the rows in turn over the grid; each thread keeps its columns' sums of
// dy n and dy, which the workgroup adds in group order and leaves in part[0 / 1][workgroup][dim].
template <int DT, int GDT, int TPR, int CH>
__global__ __launch_bounds__((ln_bwd_threads<TPR>()), 4) void layernorm_bwd_kernel(
    const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ weight, const void* dres, int rows,
    int dim, void* dx, float* __restrict__ part) {
    constexpr int NT = ln_bwd_threads<TPR>(), GROUPS = NT / TPR;
    constexpr bool SHARE = GROUPS > 1;  // several rows a workgroup: their sums meet in LDS
    __shared__ float lds[2 * 2 * (NT / 64)];
    __shared__ float s_cols[SHARE ? 2 * TPR * 8 * CH : 1];
    const int l = threadIdx.x % TPR, group = row_group<TPR>();
    const Elements<TPR, CH> el(l, dim);
    float aw[CH][8], ab[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) aw[c][j] = ab[c][j] = 0.0f;
    const float inv_dim = 1.0f / static_cast<float>(dim);
    // (with 16 elements a thread the weights are read again, from the caches, where they are used)
    constexpr bool HOLD = CH == 1;
    auto weights = [&](int c, float (&w)[8]) {
        if (weight) load8_any<NSOSX_F32>(weight, el.at[c], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = weight ? w[j] : 1.0f;
    };
    float held[8];
    if constexpr (HOLD) weights(0, held);
    int turn = 0;
    auto pass = [&](int64_t row, bool real) {
        const int64_t base = row * dim;
        Raw8<DT> xr[CH], dr[CH];
        Raw8<GDT> gr[CH];
        float mu = mean[row], q = rstd[row];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            xr[c].load(x, base + el.at[c]);
            gr[c].load(dy, base + el.at[c]);
        }
        if (dres) {
#pragma unroll
            for (int c = 0; c < CH; ++c) dr[c].load(dres, base + el.at[c]);
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float w[8];
            if constexpr (!HOLD) weights(c, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = (xr[c].get(j) - mu) * q, d = real ? gr[c].get(j) : 0.0f;
                aw[c][j] = __fmaf_rn(d, v, aw[c][j]);
                ab[c][j] += d;
                const float m = el.mine(c, j) ? d * (HOLD ? held[j] : w[j]) : 0.0f;
                s[0] += m;
                s[1] = __fmaf_rn(m, v, s[1]);
            }
        }
        if (dres && TPR > 64) {
            // dx may be dres, and a row's last two threads share elements across waves: read before any is
            // written
#pragma unroll
            for (int c = 0; c < CH; ++c) dr[c].wait();
        }
        row_sums<TPR, 2, NT>(s, lds, turn++);
        if (!real) return;
        const float m1 = s[0] * inv_dim, m2 = s[1] * inv_dim;
        asm volatile("" : "+v"(mu), "+v"(q));  // (both are formed again, not kept in registers)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float o[8], w[8];
            if constexpr (!HOLD) weights(c, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[j] = q * (gr[c].get(j) * (HOLD ? held[j] : w[j]) - m1 - (xr[c].get(j) - mu) * q * m2);
                if (dres) o[j] += dr[c].get(j);
            }
            if (el.any(c)) store8_any<DT>(dx, base + el.at[c], o);
        }
    };
    int64_t r0 = (int64_t)blockIdx.x * GROUPS;
    for (; r0 + GROUPS <= rows; r0 += (int64_t)gridDim.x * GROUPS) pass(r0 + group, true);
    if (r0 < rows) pass(min(r0 + group, (int64_t)rows - 1), r0 + group < rows);
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
                        // (element j of lane l at j * TPR + l: a wave's lanes on banks of their own; what
                        // the tail's threads hold twice is the same sums)
                        const int e = (c * 8 + j) * TPR + l;
                        sw[e] = k ? sw[e] + aw[c][j] : aw[c][j];
                        sb[e] = k ? sb[e] + ab[c][j] : ab[c][j];
                    }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < dim; e += NT) {
            // the last piece's tail lies with the thread whose elements end the row
            int p = e / 8, j = e % 8;
            if (p * 8 > dim - 8) j = e - (dim - 8);
            const int at = (p / TPR * 8 + j) * TPR + p % TPR;
            pw[e] = sw[at];
            pb[e] = sb[at];
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (el.any(c)) {
                store8_any<NSOSX_F32>(pw, el.at[c], aw[c]);
                store8_any<NSOSX_F32>(pb, el.at[c], ab[c]);
            }
    }
}

// Rows past kLnRegDim (and below 8): dx with a workgroup per row, in two readings of it.
template <int DT, int GDT, int NT>
__global__ __launch_bounds__(NT) void layernorm_bwd_long_kernel(
    const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ weight, const void* dres, int dim,
    void* dx) {
    __shared__ float lds[2 * 2 * (NT / 64)];
    const int64_t base = (int64_t)blockIdx.x * dim;
    const float mu = mean[blockIdx.x], q = rstd[blockIdx.x];
    float s[2] = {0.0f, 0.0f};
    for (int e = threadIdx.x; e < dim; e += NT) {
        const float n = (load_act<DT>(x, base + e) - mu) * q;
        const float g = load_act<GDT>(dy, base + e) * (weight ? weight[e] : 1.0f);
        s[0] += g;
        s[1] = __fmaf_rn(g, n, s[1]);
    }
    row_sums<NT, 2, NT>(s, lds, 0);
    const float inv_dim = 1.0f / static_cast<float>(dim);
    const float m1 = s[0] * inv_dim, m2 = s[1] * inv_dim;
    for (int e = threadIdx.x; e < dim; e += NT) {
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

// out0[c], out1[c] = the sums over n rows of part[0], part[1] (a NULL out is skipped), in a fixed order.
// 16 columns a workgroup (64 B of a row) at a time, a row of partial sums per 16 lanes: enough workgroups for
// every load to be on its way at once.  Each thread adds its rows in order, the threads as a tree.
constexpr int kLnSumWorkgroups = 1 << 16;  // past a million columns each takes several sixteens: a launch ends at 2^32 threads

__global__ __launch_bounds__(1024) void column_sums_kernel(const float* __restrict__ part, int n,
                                                           int cols, float* out0, float* out1) {
    float* out = blockIdx.y ? out1 : out0;
    if (!out) return;
    __shared__ float s[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < cols; c0 += (int64_t)gridDim.x * 16) {
        const int64_t c = c0 + (lane & 15);
        const float* p = part + (int64_t)blockIdx.y * n * cols + min(c, (int64_t)cols - 1);
        float sum = 0.0f;
#pragma unroll 8
        for (int r = threadIdx.x >> 4; r < n; r += 64) sum += p[(int64_t)r * cols];
        sum += lane_xor<16>(sum);
        sum += lane_xor<32>(sum);
        if (lane < 16) s[wave][lane] = sum;
        __syncthreads();
        if (threadIdx.x < 16 && c < cols) {
            for (int w = 1; w < 16; ++w) sum += s[w][lane];
            out[c] = sum;
        }
        __syncthreads();
    }
}

// Threads a row and elements a thread (8 CH): as few threads as hold the row in registers.  Add and norm
// of 67 million bf16 places: rows of 32 to 256 in a whole wave 707, 374, 206 and 119 us, in 8 to 32 threads
// 121, 92, 92 and 92; of 777, 1024 and 2048 in 256 threads 326, 160 and 106, in a wave 110, 92 and 97; of
// 4096 and 8192 in 1024 threads 171 and 114, in 256 94 and 99; rows that are read again (the kernel
// without a row in registers) 370, 340 and 305 at 4096, 8192 and 16384.
struct LnShape { int tpr, ch; };

static LnShape ln_shape(int dim) {
    if (dim <= 64) return {8, 1};
    if (dim <= 128) return {16, 1};
    if (dim <= 256) return {32, 1};
    if (dim <= 2048) return {64, (dim + 511) / 512};
    if (dim <= 8192) return {256, (dim + 2047) / 2048};
    return {1024, 2};
}

// ... of the gradients, whose threads hold three rows' pieces and two sums of them: 8 elements each
// (16 past 8192, where a workgroup takes a row)
static LnShape ln_bwd_shape(int dim) {
    int tpr = 8;
    while (tpr < 1024 && tpr * 8 < dim) tpr *= 2;
    return {tpr, tpr * 8 < dim ? 2 : 1};
}

#define NSOSX_LN_BWD_SHAPES(GO)                                                                 \
    switch (sh.tpr * sh.ch) {                                                                   \
        case 8: GO(8, 1); break;                                                                \
        case 16: GO(16, 1); break;                                                              \
        case 32: GO(32, 1); break;                                                              \
        case 64: GO(64, 1); break;                                                              \
        case 128: GO(128, 1); break;                                                            \
        case 256: GO(256, 1); break;                                                            \
        case 512: GO(512, 1); break;                                                            \
        case 1024: GO(1024, 1); break;                                                          \
        default: GO(1024, 2); break;                                                            \
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
    return (int64_t)rows * (dim > kLnRegDim ? 1024 : dim < 8 ? 64 : ln_shape(dim).tpr) + 1024;
}

constexpr int kLnWorkgroups = 512;  // of the gradients at most: each leaves a row of partial sums

static int ln_bwd_workgroups(int rows, int dim) {
    if (dim > kLnRegDim || dim < 8) return rows < 64 ? rows : 64;
    const int tpr = ln_bwd_shape(dim).tpr, groups = tpr > kLnBwdThreads ? 1 : kLnBwdThreads / tpr;
    const int need = (rows + groups - 1) / groups;
    const int most = tpr > kLnBwdThreads ? kLnWorkgroups / 2 : kLnWorkgroups;  // (one a CU, else two)
    return need < most ? need : most;
}

template <int DT, int ODT>
static void launch_layernorm(const void* x, const void* delta, const float* weight,
                             const float* bias, int rows, int dim, float eps, void* sum, void* y,
                             float* mean, float* rstd, hipStream_t st) {
    if (dim > kLnRegDim || dim < 8) {
#define NSOSX_LN(NT)                                                                                      \
    hipLaunchKernelGGL((layernorm_long_kernel<DT, ODT, NT>), dim3(rows), dim3(NT), 0, st, x, delta, weight, \
                       bias, dim, eps, sum, y, mean, rstd)
        if (dim < 8) NSOSX_LN(64);
        else NSOSX_LN(1024);
#undef NSOSX_LN
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
    if (dim > kLnRegDim || dim < 8) {
#define NSOSX_LN(NT)                                                                                       \
    hipLaunchKernelGGL((layernorm_bwd_long_kernel<DT, GDT, NT>), dim3(rows), dim3(NT), 0, st, dy, x, mean, \
                       rstd, weight, dres, dim, dx)
        if (dim < 8) NSOSX_LN(64);
        else NSOSX_LN(1024);
#undef NSOSX_LN
        if (part)
            hipLaunchKernelGGL((layernorm_cols_kernel<DT, GDT>), dim3((dim - 1) / 256 + 1, wgs),
                               dim3(256), 0, st, dy, x, mean, rstd, rows, dim, part);
        return;
    }
    const LnShape sh = ln_bwd_shape(dim);
    const dim3 grid(wgs), block(sh.tpr > kLnBwdThreads ? sh.tpr : kLnBwdThreads);
#define NSOSX_LN(T, C)                                                                             \
    hipLaunchKernelGGL((layernorm_bwd_kernel<DT, GDT, T, C>), grid, block, 0, st, dy, x, mean, rstd, \
                       weight, dres, rows, dim, dx, part)
    NSOSX_LN_BWD_SHAPES(NSOSX_LN)
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
    if (cols) {
        const int wgs = (dim - 1) / 16 + 1;
        hipLaunchKernelGGL(column_sums_kernel, dim3(wgs < kLnSumWorkgroups ? wgs : kLnSumWorkgroups, 2), dim3(1024), 0, st,
                           part, ln_bwd_workgroups(rows, dim), dim, dweight, dbias);
    }
    return check_launch("layernorm_backward");
}
