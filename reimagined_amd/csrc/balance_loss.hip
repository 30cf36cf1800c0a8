// The router's balance loss, per-expert counts and its gradient on gfx950.  With p the
// normalised scores of a row (softmax, or sigmoids over their sum), N_s the valid rows of sequence
// s, M the sequences that have any, and count_se the choices of expert e in s:
//   loss = 1/M sum_s E sum_e (count_se / (k N_s)) (sum_r p_re / N_s)
//   dloss/dx_rj = E / (M k N_s^2) p_rj (count_sj - sum_e count_se p_re)  [(1 - sigmoid) for sigmoids]
// Sixteen lanes per row, as in the scored routing, four neighbouring columns a load: the row's sums are
// four lane exchanges, and one read of the logits is all either pass does.  Both are bound by latency up
// to some ten thousand rows: 16384 x 256 f32 sigmoids, k 8, take 8.6 us for the blocks' sums, 7.6 to add
// them up (a chain of loads, barriers and one atomic) and 10.7 back (34 MB read and written: 3.1 TB/s).
// With a scalar load a column they took 13, 14 and 15, with one workgroup a sequence to add them up 14.
// Both passes look through all sequences' bounds in each of their workgroups (512 and rows / 16 of them): for
// batches of up to some thousand sequences.
#include "train.hpp"

namespace nsosx {

constexpr int kBalRows = 64;  // of a step of the forward pass: all of them in flight at once
constexpr int kBalBlocks = 512;  // two a CU; more rows take more steps each (1000000 x 64: 201 us without, 76 so)
constexpr int kBalMaxE = 512, kBalMaxK = 16;
constexpr int64_t kBalArrivals = 128;  // more parts of the loss are added by a launch of its own
constexpr int kBalCols = 16;  // columns of a workgroup that adds the blocks' sums
constexpr float kLog2e = 1.44269504088896340736f;

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

// V neighbouring columns, at any alignment.
template <int DT, int V> struct Cols;
template <> struct Cols<NSOSX_F32, 4> { struct __attribute__((packed, aligned(4))) T { float v[4]; }; };
template <> struct Cols<NSOSX_BF16, 4> { struct __attribute__((packed, aligned(2))) T { uint32_t v[2]; }; };

template <int DT, int V>
__device__ __forceinline__ void load_cols(const void* p, int64_t i, float (&f)[V]) {
    if constexpr (V == 1) {
        f[0] = load_act<DT>(p, i);
    } else if constexpr (DT == NSOSX_F32) {
        const auto t = *reinterpret_cast<const typename Cols<DT, V>::T*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = t.v[v];
    } else {
        const auto t = *reinterpret_cast<const typename Cols<DT, V>::T*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int v = 0; v < V; ++v)
            f[v] = __uint_as_float(v & 1 ? t.v[v / 2] & 0xffff0000u : t.v[v / 2] << 16);
    }
}

template <int DT, int V>
__device__ __forceinline__ void store_cols(void* p, int64_t i, const float (&f)[V]) {
    if constexpr (V == 1) {
        store_act<DT>(p, i, f[0]);
    } else {
        typename Cols<DT, V>::T t;
        if constexpr (DT == NSOSX_F32) {
#pragma unroll
            for (int v = 0; v < V; ++v) t.v[v] = f[v];
            *reinterpret_cast<typename Cols<DT, V>::T*>(static_cast<float*>(p) + i) = t;
        } else {
#pragma unroll
            for (int v = 0; v < V; v += 2) t.v[v / 2] = pack_bf16x2(f[v], f[v + 1]);
            *reinterpret_cast<typename Cols<DT, V>::T*>(static_cast<uint16_t*>(p) + i) = t;
        }
    }
}

// A lane's columns: NV times V of them, at[i] the first.  Those that would pass the row's end are its last
// V instead; the first skip[i] of them are another lane's and stay out of the row's sums.  (V is 1 below
// four experts.)
template <int NV, int V>
struct Lane {
    int at[NV], skip[NV];
    __device__ __forceinline__ Lane(int l, int E) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 16 + l) * V;
            at[i] = min(c, E - V);
            skip[i] = min(c - at[i], V);
        }
    }
};

template <int DT, int NV, int V>
__device__ __forceinline__ void load_row(const void* logits, int64_t base, const Lane<NV, V>& ln, float (&x)[NV][V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load_cols<DT, V>(logits, base + ln.at[i], x[i]);
}

// The row's normalised scores in place of its logits, and for sigmoids with REST their 1 - sigmoid; the
// exponential and reciprocal units, whose results are off by a few half steps.
template <int NV, int V, bool SIG, bool REST>
__device__ __forceinline__ void row_probs(const Lane<NV, V>& ln, float (&p)[NV][V], float (&rest)[NV][V]) {
    float mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) mx = fmaxf(mx, p[i][v]);
    mx = max16(mx);
    // Sigmoids of a row whose logits are all far below 0 would sum to 0: they are taken times e^-mx.
    const float shift = SIG && mx > -60.0f ? 0.0f : mx;
    const bool far = SIG && __any(shift != 0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (SIG) {
                const float e = __builtin_amdgcn_exp2f(fabsf(p[i][v]) * -kLog2e);
                const float big = __builtin_amdgcn_rcpf(1.0f + e);
                float small = e * big;
                if constexpr (REST) rest[i][v] = p[i][v] < 0.0f ? big : small;
                if (far && p[i][v] < 0.0f) small = __builtin_amdgcn_exp2f((p[i][v] - shift) * kLog2e) * big;
                p[i][v] = p[i][v] < 0.0f ? small : big;
            } else {
                p[i][v] = __builtin_amdgcn_exp2f((p[i][v] - shift) * kLog2e);
            }
            sum += v >= ln.skip[i] ? p[i][v] : 0.0f;
        }
    const float inv = 1.0f / sum16(sum);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) p[i][v] *= inv;
}

// One block of rows, a row per sixteen lanes: for each sequence in it, the sums of p and the counts, left
// in slot block + sequence (no two pairs share one: along the rows each step raises one of them or both).
template <int DT, int NV, int V, bool SIG>
__global__ __launch_bounds__(1024) void balance_sums_kernel(Balance P, int steps, float* __restrict__ part,
                                                            int32_t* __restrict__ counts,
                                                            int32_t* __restrict__ tokens,
                                                            uint32_t* __restrict__ arrived) {
    __shared__ float s_sum[16][NV * 16 * V];
    __shared__ int32_t s_count[NV * 16 * V], s_tokens, s_first, s_last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = threadIdx.x & 15;
    const int64_t r0 = (int64_t)blockIdx.x * kBalRows * steps, r1 = min(r0 + kBalRows * steps, (int64_t)P.rows);
    const Lane<NV, V> ln(l, P.E);
    float p[NV][V], rest[NV][V];
    int64_t r = 0;
    int chosen = -1;
    bool valid = false;
    auto take = [&](int64_t at) {
        r = at + (threadIdx.x >> 4);
        const int64_t rr = min(r, r1 - 1);
        valid = r < r1 && (!P.valid || P.valid[rr]);
        load_row<DT, NV, V>(P.logits, rr * P.stride, ln, p);
        chosen = valid && l < P.k ? P.selected[rr * P.k + l] : -1;
        row_probs<NV, V, SIG, false>(ln, p, rest);
    };
    if (steps == 1) take(r0);
    if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;  // of the next launch
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
        float sums[NV][V] = {};
        for (int64_t at = r0 + (lo - r0) / kBalRows * kBalRows; at < hi; at += kBalRows) {
            if (steps > 1) take(at);
            const bool in = valid && r >= lo && r < hi;
            if (in && chosen >= 0 && chosen < P.E) atomicAdd(&s_count[chosen], 1);
            if (in && l == 0) atomicAdd(&s_tokens, 1);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) sums[i][v] += in ? p[i][v] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float sum = sums[i][v];
                sum += lane_xor<16>(sum);
                sum += lane_xor<32>(sum);
                if (lane < 16) s_sum[wave][ln.at[i] + v] = sum;  // (what two lanes hold is the same)
            }
        __syncthreads();
        const int64_t slot = (int64_t)blockIdx.x + s;
        for (int e = threadIdx.x; e < P.E; e += 1024) {
            float sum = s_sum[0][e];
#pragma unroll
            for (int w = 1; w < 16; ++w) sum += s_sum[w][e];
            part[slot * P.E + e] = sum;
            counts[slot * P.E + e] = s_count[e];
        }
        if (threadIdx.x == 0) tokens[slot] = s_tokens;
        __syncthreads();
    }
}

// The loss of its parts, in a fixed order, by one workgroup.
template <int NT>
__device__ __forceinline__ void add_loss(int64_t parts, int S, const double* loss_part, const int32_t* tokens,
                                         float* __restrict__ loss) {
    __shared__ double s_loss[NT];
    __shared__ int32_t s_some[NT];
    double f = 0.0;
    int32_t some = 0;
    for (int64_t i = threadIdx.x; i < parts; i += NT)
        f += __hip_atomic_load(loss_part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = threadIdx.x; i < S; i += NT)
        some += __hip_atomic_load(tokens + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) > 0;
    s_loss[threadIdx.x] = f;
    s_some[threadIdx.x] = some;
    __syncthreads();
    for (int o = NT / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) {
            s_loss[threadIdx.x] += s_loss[threadIdx.x + o];
            s_some[threadIdx.x] += s_some[threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = s_some[0] ? (float)(s_loss[0] / s_some[0]) : 0.0f;
}

// kBalCols columns of a sequence: its blocks' sums, sixteen runs of them side by side.  The workgroup that
// arrives last adds the loss's parts, where `arrived` counts them.
__global__ __launch_bounds__(256) void balance_finish_kernel(Balance P, int64_t block_rows, const float* __restrict__ part,
                                                             const int32_t* __restrict__ pcounts,
                                                             const int32_t* __restrict__ ptokens,
                                                             int32_t* __restrict__ counts, int32_t* tokens,
                                                             float* __restrict__ mean, double* loss_part,
                                                             uint32_t* arrived, float* __restrict__ loss) {
    __shared__ float s_sum[16][kBalCols];
    __shared__ int32_t s_count[16][kBalCols], s_tokens, s_last;
    const int s = blockIdx.y;
    const int64_t lo = P.cu ? max(0, P.cu[s]) : 0, hi = P.cu ? min(P.rows, P.cu[s + 1]) : P.rows;
    const int64_t b0 = lo / block_rows, b1 = hi > lo ? (hi - 1) / block_rows + 1 : b0;
    const int l = threadIdx.x % kBalCols, run = threadIdx.x / kBalCols, e = blockIdx.x * kBalCols + l;
    float sum = 0.0f;
    int32_t count = 0, n = 0;
    if (threadIdx.x == 0) s_tokens = 0;
    __syncthreads();
    for (int64_t b = b0 + threadIdx.x; b < b1; b += 256) n += ptokens[b + s];
    if (e < P.E) {
#pragma unroll 4
        for (int64_t b = b0 + run; b < b1; b += 16) {
            sum += part[(b + s) * P.E + e];
            count += pcounts[(b + s) * P.E + e];
        }
    }
    if (n) atomicAdd(&s_tokens, n);
    s_sum[run][l] = sum;
    s_count[run][l] = count;
    __syncthreads();
    const int32_t total = s_tokens;
    if (threadIdx.x < kBalCols) {
        for (int q = 1; q < 16; ++q) {
            sum += s_sum[q][l];
            count += s_count[q][l];
        }
        const float avg = total ? sum / static_cast<float>(total) : 0.0f;
        double f = 0.0;
        if (e < P.E) {
            counts[(int64_t)s * P.E + e] = count;
            mean[(int64_t)s * P.E + e] = avg;
            f = total ? (double)count * avg * P.E / ((double)P.k * total) : 0.0;
        }
        for (int o = kBalCols / 2; o > 0; o >>= 1) f += __shfl_xor(f, o, kBalCols);
        if (l == 0) {
            const int64_t at = (int64_t)s * gridDim.x + blockIdx.x;
            __hip_atomic_store(loss_part + at, f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (blockIdx.x == 0) __hip_atomic_store(tokens + s, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = arrived && __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
                                    gridDim.x * gridDim.y - 1;
        }
    }
    __syncthreads();
    if (s_last) add_loss<256>((int64_t)gridDim.x * gridDim.y, P.S, loss_part, tokens, loss);
}

// The loss's parts where they are many: 25 ns and a write-back of an L2 for each arrival cost more than a
// launch (the forward pass of 65536 x 64 in 1500 sequences, 6000 parts: 157 us with arrivals, 31 so; 16384 x
// 256 in one, 16 parts: 15.3 and 16.1; in eight, 128 parts: 16.4 and 15.0, and 3 of host time for the launch).
__global__ __launch_bounds__(1024) void balance_loss_kernel(int64_t parts, int S, const double* loss_part,
                                                            const int32_t* tokens, float* __restrict__ loss) {
    add_loss<1024>(parts, S, loss_part, tokens, loss);
}

// Nothing to add up: no row, or no sequence.
__global__ __launch_bounds__(256) void balance_none_kernel(int S, int E, float* loss, int32_t* counts,
                                                           int32_t* tokens, float* mean) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i == 0) *loss = 0.0f;
    if (i < S) tokens[i] = 0;
    if (i < (int64_t)S * E) {
        counts[i] = 0;
        mean[i] = 0.0f;
    }
}

template <int DT, int NV, int V, bool SIG>
__global__ __launch_bounds__(256) void balance_bwd_kernel(Balance P, const int32_t* __restrict__ counts,
                                                          const int32_t* __restrict__ tokens, float scale,
                                                          const float* __restrict__ dloss, const void* add,
                                                          void* dlogits) {
    __shared__ int32_t s_seq[16], s_some;
    const int l = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t r0 = (int64_t)blockIdx.x * 16, r = r0 + group, rr = min(r, (int64_t)P.rows - 1);
    const Lane<NV, V> ln(l, P.E);
    float p[NV][V], rest[NV][V], a[NV][V];
    load_row<DT, NV, V>(P.logits, rr * P.stride, ln, p);
    if (add) load_row<DT, NV, V>(add, rr * P.E, ln, a);
    if (threadIdx.x < 16) s_seq[threadIdx.x] = P.cu ? -1 : 0;
    if (threadIdx.x == 0) s_some = 0;
    __syncthreads();
    int some = 0;
    for (int s = threadIdx.x; s < P.S; s += 256) {
        some += tokens[s] > 0;
        if (P.cu) {
            const int64_t lo = max((int64_t)P.cu[s], r0), hi = min((int64_t)P.cu[s + 1], r0 + 16);
            for (int64_t q = lo; q < hi; ++q) s_seq[q - r0] = s;
        }
    }
    if (some) atomicAdd(&s_some, some);
    __syncthreads();
    if (r >= P.rows) return;
    const int s = s_seq[group];
    const int n = s >= 0 ? tokens[s] : 0;
    float g[NV][V];
    if (n > 0 && !(P.valid && !P.valid[r])) {
        float dot = 0.0f;
        // (the p sum to 1, so a part that all counts share changes nothing but the rounding: without it the
        // difference of a balanced router's counts and their mean keeps its bits, and is 0 where they are equal)
        const int even = (int)((int64_t)P.k * n / P.E);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) g[i][v] = static_cast<float>(counts[(int64_t)s * P.E + ln.at[i] + v] - even);
        row_probs<NV, V, SIG, true>(ln, p, rest);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) dot += v >= ln.skip[i] ? g[i][v] * p[i][v] : 0.0f;
        dot = sum16(dot);
        const float nf = static_cast<float>(n);
        const float f = scale * (dloss ? *dloss : 1.0f) * static_cast<float>(P.E) /
                        (static_cast<float>(P.k) * static_cast<float>(s_some) * nf) / nf;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                g[i][v] = p[i][v] * (g[i][v] - dot) * f;
                if constexpr (SIG) g[i][v] *= rest[i][v];
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) g[i][v] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (add) {
#pragma unroll
            for (int v = 0; v < V; ++v) g[i][v] += a[i][v];
        }
        if (ln.skip[i] < V) store_cols<DT, V>(dlogits, r * P.E + ln.at[i], g[i]);
    }
}

static int64_t bal_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int bal_steps(int rows) { return (int)bal_ceil(bal_ceil(rows, kBalRows), kBalBlocks); }
static int64_t bal_blocks(int rows) { return rows > 0 ? bal_ceil(rows, (int64_t)kBalRows * bal_steps(rows)) : 0; }

#define NSOSX_BAL_NV(GO, DT, SIG)                 \
    do {                                          \
        if (p.E < 4) GO(DT, 1, 1, SIG);           \
        else if (p.E <= 64) GO(DT, 1, 4, SIG);    \
        else if (p.E <= 128) GO(DT, 2, 4, SIG);   \
        else if (p.E <= 256) GO(DT, 4, 4, SIG);   \
        else GO(DT, 8, 4, SIG);                   \
    } while (0)
#define NSOSX_BAL(GO, dtype, sig)                                                    \
    do {                                                                             \
        if ((dtype) == NSOSX_F32) {                                                  \
            if (sig) NSOSX_BAL_NV(GO, NSOSX_F32, true);                              \
            else NSOSX_BAL_NV(GO, NSOSX_F32, false);                                 \
        } else {                                                                     \
            if (sig) NSOSX_BAL_NV(GO, NSOSX_BF16, true);                             \
            else NSOSX_BAL_NV(GO, NSOSX_BF16, false);                                \
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
    if ((int64_t)p.rows * 16 + 256 > 0xffffffffLL || p.S > 65535)
        return fail(NSOSX_ERR_OVERFLOW, name + ": rows or sequences too large");
    return NSOSX_OK;
}

}  // namespace nsosx

using namespace nsosx;

// workspace: the loss's parts (f64), the arrivals (16 bytes), per slot (block + sequence) E sums, E counts
// and the rows
extern "C" int64_t nsosx_moe_balance_loss_workspace(int rows, int experts, int S) {
    if (rows < 0 || experts <= 0 || S < 0) return 0;
    const int64_t parts = (int64_t)S * ((experts + kBalCols - 1) / kBalCols);
    return parts * 8 + 16 + (bal_blocks(rows) + S) * (2 * (int64_t)experts + 1) * 4;
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
    if (reinterpret_cast<uintptr_t>(workspace) & 7)
        return fail(NSOSX_ERR_INVALID, "moe_balance_loss: workspace must be 8-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (rows == 0 || S == 0) {
        hipLaunchKernelGGL(balance_none_kernel, dim3((unsigned)(((int64_t)S * experts + 255) / 256 + 1)), dim3(256),
                           0, st, S, experts, loss, counts, tokens, mean_prob);
        return check_launch("moe_balance_loss");
    }
    const int steps = bal_steps(rows);
    const int64_t blocks = bal_blocks(rows), slots = blocks + S;
    const dim3 grid((experts + kBalCols - 1) / kBalCols, S);
    const int64_t parts = (int64_t)grid.x * S;
    const bool few = parts <= kBalArrivals;
    double* loss_part = static_cast<double*>(workspace);
    uint32_t* arrived = reinterpret_cast<uint32_t*>(loss_part + parts);
    float* part = reinterpret_cast<float*>(arrived + 4);
    int32_t* pcounts = reinterpret_cast<int32_t*>(part + slots * experts);
    int32_t* ptokens = pcounts + slots * experts;
#define NSOSX_BAL_GO(DT, NV, V, SIG)                                                                     \
    hipLaunchKernelGGL((balance_sums_kernel<DT, NV, V, SIG>), dim3((unsigned)blocks), dim3(1024), 0, st, p, \
                       steps, part, pcounts, ptokens, arrived)
    NSOSX_BAL(NSOSX_BAL_GO, logits_dtype, sigmoid);
#undef NSOSX_BAL_GO
    hipLaunchKernelGGL(balance_finish_kernel, grid, dim3(256), 0, st, p, (int64_t)kBalRows * steps, part, pcounts, ptokens,
                       counts, tokens, mean_prob, loss_part, few ? arrived : nullptr, loss);
    if (!few)
        hipLaunchKernelGGL(balance_loss_kernel, dim3(1), dim3(1024), 0, st, parts, S, loss_part, tokens, loss);
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
#define NSOSX_BAL_GO(DT, NV, V, SIG)                                                                       \
    hipLaunchKernelGGL((balance_bwd_kernel<DT, NV, V, SIG>), grid, dim3(256), 0, st, p, counts, tokens, scale, \
                       dloss, add, dlogits)
    NSOSX_BAL(NSOSX_BAL_GO, logits_dtype, sigmoid);
#undef NSOSX_BAL_GO
    return check_launch("moe_balance_loss_backward");
}
