// Gated linear recurrence over packed ragged batches, its gradients and its single-token step, on
// gfx950.  Per channel, with sr = sigmoid(rg), s = sigmoid(ig):
//   g = rate softplus(lam) sr,  a = exp(-g),  beta = sqrt(1 - a^2),  h_t = a_t h_(t-1) + beta_t s_t x_t
// The tokens of the whole batch are one stream, cut into tiles of kTile tokens whatever the sequences'
// lengths: a token that starts a sequence takes h from that sequence's initial state instead of from the
// token before it, so no tile knows or waits for the longest sequence.
// A tile's effect on what enters it is h -> A h + H, with A the product of its decays (0 where a
// sequence starts inside); the tiles' pairs (A, H) give every tile the state that enters it.
// Backwards the same stream runs the other way in m_t = a_t dh_t, dh_t = dy_t + m_(t+1): a sequence's
// last token takes dfinal in place of m_(t+1), its first token's m is dinitial.  h is formed again
// from the forward's states at the tiles' borders (f32, one per kTile tokens), so y is not read.
#include "train.hpp"

#include <cmath>

namespace nsosx {

constexpr int kTile = 128;      // tokens; the distance of the kept states
constexpr int kRecMaxDim = 1 << 30;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Two neighbouring channels of a token (one where D is 1), as loaded.
template <int DT, int V> struct Pair;
template <> struct Pair<NSOSX_BF16, 2> {
    uint32_t w;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        w = reinterpret_cast<const bf16x2_any*>(static_cast<const uint16_t*>(p) + i)->w;
    }
    __device__ __forceinline__ float get(int k) const {
        return __uint_as_float(k ? w & 0xffff0000u : w << 16);
    }
};
template <> struct Pair<NSOSX_F32, 2> {
    float v[2];
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        const f32x2_any a = *reinterpret_cast<const f32x2_any*>(static_cast<const float*>(p) + i);
        v[0] = a.v[0];
        v[1] = a.v[1];
    }
    __device__ __forceinline__ float get(int k) const { return v[k]; }
};
template <int DT> struct Pair<DT, 1> {
    float v;
    __device__ __forceinline__ void load(const void* p, int64_t i) { v = load_act<DT>(p, i); }
    __device__ __forceinline__ float get(int) const { return v; }
};

template <int DT, int V>
__device__ __forceinline__ void store_pair(void* p, int64_t i, const float (&v)[V]) {
    if constexpr (V == 1) {
        store_act<DT>(p, i, v[0]);
    } else if constexpr (DT == NSOSX_F32) {
        f32x2_any a;
        a.v[0] = v[0];
        a.v[1] = v[1];
        *reinterpret_cast<f32x2_any*>(static_cast<float*>(p) + i) = a;
    } else {
        bf16x2_any a;
        a.w = pack_bf16x2(v[0], v[1]);
        *reinterpret_cast<bf16x2_any*>(static_cast<uint16_t*>(p) + i) = a;
    }
}

// 1 / (1 + e^-x) on the exponential and reciprocal units: off by up to (5 + 2 |x|) half steps.
__device__ __forceinline__ float sigmoid_fast(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e));
}

// ... and 1 - sigmoid(x) without the cancellation of large x (e^-|x| cannot overflow)
__device__ __forceinline__ void sigmoid_both(float x, float& s, float& rest) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * -kLog2e);
    const float p = __builtin_amdgcn_rcpf(1.0f + e), n = e * p;
    s = x < 0.0f ? n : p;
    rest = x < 0.0f ? p : n;
}

// rate softplus(lam) in units of log 2: a = 2^(-k2 sr)
__device__ __forceinline__ float decay_rate(float lam, float rate) {
    return rate * (fmaxf(lam, 0.0f) + log1pf(expf(-fabsf(lam)))) * kLog2e;
}

// a and p = 1 - a^2 from q = -log2(a).  Where a is near 1 the difference would cancel: below
// t = -log(a^2) = 0.5 it is t times a fit of (1 - e^-t) / t (own least-squares fit, relative error
// 2e-9 before rounding); above, 1 - a^2 is exact to 2e-7.
__device__ __forceinline__ void decay(float q, float& a, float& p) {
    a = __builtin_amdgcn_exp2f(-q);
    const float t = q * (2.0f * kLn2);
    float f = __fmaf_rn(t, -0.0011216349f, 0.008187386f);
    f = __fmaf_rn(t, f, -0.04162909f);
    f = __fmaf_rn(t, f, 0.16666225f);
    f = __fmaf_rn(t, f, -0.49999982f);
    f = __fmaf_rn(t, f, 1.0f);
    p = t < 0.5f ? t * f : __fmaf_rn(-a, a, 1.0f);
}

// Where the tile's sequences start and end: s_start[i] / s_end[i] hold the sequence whose first /
// last token is token i of the tile, else -1.  Every workgroup reads all of cu_seqlens, a few loads
// that do not depend on each other, rather than search it in log2(S) that do.
template <int NT>
__device__ __forceinline__ void tile_borders(const int32_t* __restrict__ cu, int S, int64_t t0,
                                             int32_t* s_start, int32_t* s_end) {
    for (int i = threadIdx.x; i < kTile; i += NT) s_start[i] = s_end[i] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < S; s += NT) {
        const int64_t lo = cu[s], hi = cu[s + 1];
        if (hi <= lo) continue;
        if (lo >= t0 && lo < t0 + kTile) s_start[lo - t0] = s;
        if (hi > t0 && hi <= t0 + kTile) s_end[hi - 1 - t0] = s;
    }
    __syncthreads();
}

// A bit per token of this wave's R: starts, ends, and tokens of some sequence.
template <int R>
__device__ __forceinline__ void wave_masks(const int32_t* s_start, const int32_t* s_end, int wave,
                                           int64_t t0, int64_t lo, int64_t hi, uint32_t& starts,
                                           uint32_t& ends, uint32_t& inside) {
    const int lane = threadIdx.x & 63;
    const int i = wave * R + min(lane, R - 1);
    const int64_t t = t0 + i;
    starts = (uint32_t)__ballot(lane < R && s_start[i] >= 0);
    ends = (uint32_t)__ballot(lane < R && s_end[i] >= 0);
    inside = (uint32_t)__ballot(lane < R && t >= lo && t < hi);
}

// What an empty sequence leaves: its initial state (or zeros), both ways.
template <int V, int NT>
__device__ __forceinline__ void empty_states(const int32_t* __restrict__ cu, int S, int64_t D, int64_t ch,
                                             bool act, const float* __restrict__ from,
                                             float* __restrict__ to) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int s0 = wave * 64; s0 < S; s0 += NT) {
        const int s = s0 + lane;
        uint64_t none = __ballot(s < S && cu[min(s, S - 1) + 1] <= cu[min(s, S - 1)]);
        for (; none; none &= none - 1) {
            const int64_t at = (int64_t)(s0 + __builtin_ctzll(none)) * D + ch;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (act) to[at + k] = from ? from[at + k] : 0.0f;
        }
    }
}

struct RecFwd {
    const void *x, *rg, *ig;
    int64_t xs, rs, is;  // row strides, elements
    const float* lam;
    float rate;
    const int32_t* cu;
    int S, T, D, rest;  // rest: rows of no sequence are written as zeros
    const float* initial;
    void* y;
    int64_t ys;
    float *final, *carry;  // carry [tiles, D]: the state that enters a tile
    float2* agg;           // [tiles, D]: (A, H)
};

// PASS 0 leaves the tile's (A, H); PASS 1 runs it from the state that enters it.  A workgroup takes
// 128 channels, two a lane; each wave takes R of the tile's tokens.
template <int DT, int V, int R, int PASS>
__global__ __launch_bounds__(64 * (kTile / R)) void recurrence_kernel(RecFwd P) {
    constexpr int WAVES = kTile / R, NT = 64 * WAVES;
    __shared__ int32_t s_start[kTile], s_end[kTile];
    __shared__ float s_k2[64 * V], s_a[WAVES][V][64], s_h[WAVES][V][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (P.D - 1) / (64 * V) + 1;
    const int64_t tile = blockIdx.x / blocks;
    const int64_t c0 = (int64_t)(blockIdx.x % blocks) * 64 * V, t0 = tile * kTile;
    // past the last channel: the last ones again, whose lanes compute and store the same values
    const int64_t ch = min(c0 + lane * V, (int64_t)P.D - V);
    const int64_t cb = min(c0, (int64_t)P.D - V);
    const bool act = c0 + lane * V < P.D;
    const float zero[V] = {};
    Pair<DT, V> x[R], r[R], g[R];
    const int64_t tw = t0 + wave * R;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int64_t t = min(tw + j, (int64_t)P.T - 1);
        r[j].load(P.rg, t * P.rs + ch);
        g[j].load(P.ig, t * P.is + ch);
        x[j].load(P.x, t * P.xs + ch);
    }
    for (int i = threadIdx.x; i < 64 * V; i += NT)
        s_k2[i] = decay_rate(P.lam[min(cb + i, (int64_t)P.D - 1)], P.rate);
    tile_borders<NT>(P.cu, P.S, t0, s_start, s_end);
    uint32_t starts, ends, inside;
    wave_masks<R>(s_start, s_end, wave, t0, P.cu[0], min(P.cu[P.S], P.T), starts, ends, inside);
    float a[R][V], u[R][V], k2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) k2[k] = s_k2[ch - cb + k];
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float p;
            decay(k2[k] * sigmoid_fast(r[j].get(k)), a[j][k], p);
            u[j][k] = __builtin_amdgcn_sqrtf(p) * sigmoid_fast(g[j].get(k)) * x[j].get(k);
        }
    float A[V], H[V];
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (starts >> j & 1) {
            const float* h0 = P.initial ? P.initial + (int64_t)s_start[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
            for (int k = 0; k < V; ++k) H[k] = h0 ? h0[k] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
            A[k] = starts >> j & 1 ? 0.0f : A[k] * a[j][k];
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s_a[wave][k][lane] = A[k], s_h[wave][k][lane] = H[k];
    __syncthreads();
    if constexpr (PASS == 0) {
        if (wave == 0 && act) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                A[k] = 1.0f, H[k] = 0.0f;
                for (int w = 0; w < WAVES; ++w) {
                    const float aw = s_a[w][k][lane];
                    H[k] = aw == 0.0f ? s_h[w][k][lane] : __fmaf_rn(aw, H[k], s_h[w][k][lane]);
                    A[k] = aw == 0.0f ? 0.0f : A[k] * aw;
                }
                P.agg[tile * P.D + ch + k] = make_float2(A[k], H[k]);
            }
        }
    } else {
        float h[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            h[k] = P.carry[tile * P.D + ch + k];
            for (int w = 0; w < wave; ++w) {
                const float aw = s_a[w][k][lane];
                h[k] = aw == 0.0f ? s_h[w][k][lane] : __fmaf_rn(aw, h[k], s_h[w][k][lane]);
            }
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int64_t t = tw + j;
            if (!(inside >> j & 1)) {
                if (P.rest && t < P.T && act) store_pair<DT, V>(P.y, t * P.ys + ch, zero);
                continue;
            }
            if (starts >> j & 1) {
                const float* h0 = P.initial ? P.initial + (int64_t)s_start[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] = h0 ? h0[k] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = __fmaf_rn(a[j][k], h[k], u[j][k]);
            if (act) store_pair<DT, V>(P.y, t * P.ys + ch, h);
            if ((ends >> j & 1) && P.final && act) {
                float* to = P.final + (int64_t)s_end[wave * R + j] * P.D + ch;
#pragma unroll
                for (int k = 0; k < V; ++k) to[k] = h[k];
            }
        }
        if (tile == 0 && P.final) empty_states<V, NT>(P.cu, P.S, P.D, ch, act, P.initial, P.final);
    }
}

// The state that enters every tile, from the tiles' pairs in order (reversed for the gradients).
__global__ __launch_bounds__(64) void recurrence_carry_kernel(const float2* __restrict__ agg, int tiles,
                                                              int D, int reverse,
                                                              float* __restrict__ carry) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= D) return;
    float h = 0.0f;
    for (int i = 0; i < tiles; ++i) {
        const int64_t at = (int64_t)(reverse ? tiles - 1 - i : i) * D + c;
        const float2 p = agg[at];
        carry[at] = h;
        h = p.x == 0.0f ? p.y : __fmaf_rn(p.x, h, p.y);
    }
}

struct RecBwd {
    const void *dy, *x, *rg, *ig;
    int64_t dys, xs, rs, is;
    const float* lam;
    float rate;
    const int32_t* cu;
    int S, T, D, rest;
    const float *initial, *carry, *dfinal;
    void *dx, *drg, *dig;
    int64_t dxs, drs, dis;
    float *dinitial, *dlam_part;  // dlam_part [tiles, D]
    float2* agg;                  // [tiles, D]: (A, M) of the reversed stream
    float* mcarry;                // [tiles, D]: the m that enters a tile from behind
};

template <int DT, int V, int R, int PASS>
__global__ __launch_bounds__(64 * (kTile / R)) void recurrence_bwd_kernel(RecBwd P) {
    constexpr int WAVES = kTile / R, NT = 64 * WAVES;
    __shared__ int32_t s_start[kTile], s_end[kTile];
    __shared__ float s_k2[64 * V], s_a[WAVES][V][64], s_h[WAVES][V][64], s_b[WAVES][V][64],
        s_m[WAVES][V][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (P.D - 1) / (64 * V) + 1;
    const int64_t tile = blockIdx.x / blocks;
    const int64_t c0 = (int64_t)(blockIdx.x % blocks) * 64 * V, t0 = tile * kTile;
    const int64_t ch = min(c0 + lane * V, (int64_t)P.D - V);
    const int64_t cb = min(c0, (int64_t)P.D - V);
    const bool act = c0 + lane * V < P.D;
    const float zero[V] = {};
    Pair<DT, V> x[R], r[R], g[R], d[R];
    const int64_t tw = t0 + wave * R;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int64_t t = min(tw + j, (int64_t)P.T - 1);
        r[j].load(P.rg, t * P.rs + ch);
        d[j].load(P.dy, t * P.dys + ch);
        if constexpr (PASS == 1) {
            g[j].load(P.ig, t * P.is + ch);
            x[j].load(P.x, t * P.xs + ch);
        }
    }
    for (int i = threadIdx.x; i < 64 * V; i += NT)
        s_k2[i] = decay_rate(P.lam[min(cb + i, (int64_t)P.D - 1)], P.rate);
    tile_borders<NT>(P.cu, P.S, t0, s_start, s_end);
    uint32_t starts, ends, inside;
    wave_masks<R>(s_start, s_end, wave, t0, P.cu[0], min(P.cu[P.S], P.T), starts, ends, inside);
    float k2[V], a[R][V], u[R][V];
#pragma unroll
    for (int k = 0; k < V; ++k) k2[k] = s_k2[ch - cb + k];
    float A[V], H[V], B[V], M[V];
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = B[k] = 1.0f, H[k] = M[k] = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (PASS == 1 && (starts >> j & 1)) {
            const float* h0 = P.initial ? P.initial + (int64_t)s_start[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
            for (int k = 0; k < V; ++k) H[k] = h0 ? h0[k] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float p;
            decay(k2[k] * sigmoid_fast(r[j].get(k)), a[j][k], p);
            if constexpr (PASS == 1) {
                u[j][k] = __builtin_amdgcn_sqrtf(p) * sigmoid_fast(g[j].get(k)) * x[j].get(k);
                H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
                A[k] = starts >> j & 1 ? 0.0f : A[k] * a[j][k];
            }
        }
    }
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
        if (ends >> j & 1) {
            const float* df = P.dfinal ? P.dfinal + (int64_t)s_end[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
            for (int k = 0; k < V; ++k) M[k] = df ? df[k] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            M[k] = inside >> j & 1 ? a[j][k] * (d[j].get(k) + M[k]) : 0.0f;
            B[k] = (ends >> j & 1) || !(inside >> j & 1) ? 0.0f : B[k] * a[j][k];
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        s_a[wave][k][lane] = A[k], s_h[wave][k][lane] = H[k];
        s_b[wave][k][lane] = B[k], s_m[wave][k][lane] = M[k];
    }
    __syncthreads();
    if constexpr (PASS == 0) {
        if (wave == 0 && act) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                B[k] = 1.0f, M[k] = 0.0f;
                for (int w = WAVES - 1; w >= 0; --w) {
                    const float bw = s_b[w][k][lane];
                    M[k] = bw == 0.0f ? s_m[w][k][lane] : __fmaf_rn(bw, M[k], s_m[w][k][lane]);
                    B[k] = bw == 0.0f ? 0.0f : B[k] * bw;
                }
                P.agg[tile * P.D + ch + k] = make_float2(B[k], M[k]);
            }
        }
    } else {
        float h[V], m[V], e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            h[k] = P.carry[tile * P.D + ch + k];
            for (int w = 0; w < wave; ++w) {
                const float aw = s_a[w][k][lane];
                h[k] = aw == 0.0f ? s_h[w][k][lane] : __fmaf_rn(aw, h[k], s_h[w][k][lane]);
            }
            m[k] = P.mcarry[tile * P.D + ch + k];
            for (int w = WAVES - 1; w > wave; --w) {
                const float bw = s_b[w][k][lane];
                m[k] = bw == 0.0f ? s_m[w][k][lane] : __fmaf_rn(bw, m[k], s_m[w][k][lane]);
            }
            e[k] = 0.0f;
        }
        // u becomes the state before each token
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (starts >> j & 1) {
                const float* h0 = P.initial ? P.initial + (int64_t)s_start[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] = h0 ? h0[k] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float before = h[k];
                h[k] = __fmaf_rn(a[j][k], h[k], u[j][k]);
                u[j][k] = before;
            }
        }
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            const int64_t t = tw + j;
            if (!(inside >> j & 1)) {
                if (P.rest && t < P.T && act) {
                    store_pair<DT, V>(P.dx, t * P.dxs + ch, zero);
                    store_pair<DT, V>(P.drg, t * P.drs + ch, zero);
                    store_pair<DT, V>(P.dig, t * P.dis + ch, zero);
                }
                continue;
            }
            if (ends >> j & 1) {
                const float* df = P.dfinal ? P.dfinal + (int64_t)s_end[wave * R + j] * P.D + ch : nullptr;
#pragma unroll
                for (int k = 0; k < V; ++k) m[k] = df ? df[k] : 0.0f;
            }
            float ox[V], orr[V], oi[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float sr, nr, si, ni, a2, p;
                sigmoid_both(r[j].get(k), sr, nr);
                sigmoid_both(g[j].get(k), si, ni);
                const float q = k2[k] * sr;
                decay(q, a2, p);
                const float beta = __builtin_amdgcn_sqrtf(p), xv = x[j].get(k);
                const float dh = d[j].get(k) + m[k], dg = q * kLn2;  // dg: g itself
                // g a^2 / beta goes to sqrt(g / 2) as the gate closes, and to 0 with it
                const float bent = beta > 0.0f ? dg * a[j][k] * a[j][k] * __builtin_amdgcn_rcpf(beta) : 0.0f;
                const float ev = dh * (si * xv * bent - a[j][k] * dg * u[j][k]);
                ox[k] = dh * beta * si;
                oi[k] = ox[k] * xv * ni;
                orr[k] = ev * nr;
                e[k] += ev;
                m[k] = a[j][k] * dh;
            }
            if (act) {
                store_pair<DT, V>(P.dx, t * P.dxs + ch, ox);
                store_pair<DT, V>(P.drg, t * P.drs + ch, orr);
                store_pair<DT, V>(P.dig, t * P.dis + ch, oi);
            }
            if ((starts >> j & 1) && P.dinitial && act) {
                float* to = P.dinitial + (int64_t)s_start[wave * R + j] * P.D + ch;
#pragma unroll
                for (int k = 0; k < V; ++k) to[k] = m[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) s_a[wave][k][lane] = e[k];
        __syncthreads();
        if (wave == 0 && act) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                for (int w = 1; w < WAVES; ++w) e[k] += s_a[w][k][lane];
                P.dlam_part[tile * P.D + ch + k] = e[k];
            }
        }
        if (tile == 0 && P.dinitial) empty_states<V, NT>(P.cu, P.S, P.D, ch, act, P.dfinal, P.dinitial);
    }
}

// dlam = sigmoid(lam) / softplus(lam) * sum_t e: the tiles' sums in a fixed order (64 channels a
// workgroup, its 16 waves take every 16th tile).
__global__ __launch_bounds__(1024) void recurrence_dlam_kernel(const float* __restrict__ part, int tiles,
                                                               int D, const float* __restrict__ lam,
                                                               float* __restrict__ dlam) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float sum = 0.0f;
    if (c < D)
        for (int i = wave; i < tiles; i += 16) sum += part[(int64_t)i * D + c];
    s[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || c >= D) return;
    for (int w = 1; w < 16; ++w) sum += s[w][lane];
    // sigmoid / softplus goes to 1 as both go to e^lam
    const float l = lam[c], en = expf(-fabsf(l));
    const float sig = l < 0.0f ? en / (1.0f + en) : 1.0f / (1.0f + en);
    const float sp = fmaxf(l, 0.0f) + log1pf(en);
    dlam[c] = sum * (sp == 0.0f ? 1.0f : sig / sp);
}

// One token per row: a thread per channel and run of kStepRows rows.
constexpr int kStepRows = 4;

template <int DT>
__global__ __launch_bounds__(256) void recurrence_step_kernel(
    const void* __restrict__ x, int64_t xs, const void* __restrict__ rg, int64_t rs,
    const void* __restrict__ ig, int64_t is, const float* __restrict__ lam, float rate, int rows, int D,
    const float* state, float* state_out, void* __restrict__ y, int64_t ys) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    const float k2 = decay_rate(lam[c], rate);
    for (int j = 0; j < kStepRows; ++j) {
        const int64_t r = (int64_t)blockIdx.y * kStepRows + j;
        if (r >= rows) return;
        float a, p;
        decay(k2 * sigmoid_fast(load_act<DT>(rg, r * rs + c)), a, p);
        const float u = __builtin_amdgcn_sqrtf(p) * sigmoid_fast(load_act<DT>(ig, r * is + c)) *
                        load_act<DT>(x, r * xs + c);
        const float h = __fmaf_rn(a, state[r * D + c], u);
        state_out[r * D + c] = h;
        store_act<DT>(y, r * ys + c, h);
    }
}

static int64_t rec_tiles(int64_t T) { return (T + kTile - 1) / kTile; }

// [rows, D] views of row stride (elements): whether two of them share an element.  Views of one row
// stride may lie side by side in the same rows.
static bool views_cross(const void* a, int64_t as, const void* b, int64_t bs, int64_t rows, int64_t D,
                        int64_t size) {
    if (!a || !b || rows <= 0) return false;
    const int64_t an = ((rows - 1) * as + D) * size, bn = ((rows - 1) * bs + D) * size;
    if (!overlaps(a, an, b, bn)) return false;
    if (as != bs || rows == 1) return true;
    const int64_t row = as * size;
    int64_t off = (static_cast<const char*>(b) - static_cast<const char*>(a)) % row;
    if (off < 0) off += row;
    return off < D * size || off + D * size > row;
}

static const char* rec_check(int S, int64_t T, int D, int dtype, float rate) {
    if (S < 0 || T < 0 || D <= 0) return "need sequences >= 0, tokens >= 0 and dim > 0";
    if (!valid_dtype(dtype)) return "bad dtype";
    if (!(rate > 0.0f) || rate > 3.0e38f) return "rate must be finite and > 0";
    return nullptr;
}

template <int DT, int V>
static void launch_recurrence(const RecFwd& p, hipStream_t st) {
    const int64_t tiles = rec_tiles(p.T);
    const int blocks = (p.D - 1) / (64 * V) + 1;
    const dim3 grid((unsigned)(tiles * blocks)), block(64 * (kTile / 16));
    hipLaunchKernelGGL((recurrence_kernel<DT, V, 16, 0>), grid, block, 0, st, p);
    hipLaunchKernelGGL(recurrence_carry_kernel, dim3((p.D + 63) / 64), dim3(64), 0, st, p.agg, (int)tiles,
                       p.D, 0, p.carry);
    hipLaunchKernelGGL((recurrence_kernel<DT, V, 16, 1>), grid, block, 0, st, p);
}

template <int DT, int V>
static void launch_recurrence_bwd(const RecBwd& p, hipStream_t st) {
    const int64_t tiles = rec_tiles(p.T);
    const int blocks = (p.D - 1) / (64 * V) + 1;
    const dim3 grid((unsigned)(tiles * blocks)), block(64 * (kTile / 16));
    hipLaunchKernelGGL((recurrence_bwd_kernel<DT, V, 16, 0>), grid, block, 0, st, p);
    hipLaunchKernelGGL(recurrence_carry_kernel, dim3((p.D + 63) / 64), dim3(64), 0, st, p.agg, (int)tiles,
                       p.D, 1, p.mcarry);
    hipLaunchKernelGGL((recurrence_bwd_kernel<DT, V, 16, 1>), grid, block, 0, st, p);
}

// No token: every sequence is empty, its final state is its initial one.
__global__ __launch_bounds__(256) void recurrence_empty_kernel(const float* __restrict__ from, int64_t n,
                                                               float* __restrict__ to) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.0f;
}

static void launch_empty(const float* from, int64_t n, float* to, hipStream_t st) {
    if (n > 0)
        hipLaunchKernelGGL(recurrence_empty_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st,
                           from, n, to);
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int nsosx_gated_recurrence_tile(void) { return kTile; }

extern "C" int64_t nsosx_gated_recurrence_workspace(int T, int D) {
    if (T <= 0 || D <= 0) return 0;
    return rec_tiles(T) * D * 12;
}

extern "C" int nsosx_gated_recurrence(const void* x, int64_t x_stride, const void* rg, int64_t rg_stride,
                                      const void* ig, int64_t ig_stride, const float* lam, float rate,
                                      const int32_t* cu_seqlens, int S, int T, int D, int act_dtype,
                                      const float* initial_state, int zero_rest, void* y,
                                      int64_t y_stride, float* final_state, float* carry,
                                      void* workspace, void* stream) {
    if (const char* why = rec_check(S, T, D, act_dtype, rate))
        return fail(NSOSX_ERR_INVALID, std::string("gated_recurrence: ") + why);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t sd = (int64_t)S * D;
    if (D > kRecMaxDim || sd > 0xffffffffLL - 256 ||
        rec_tiles(T) * ((D + 63) / 64) > 0xffffffffLL / 1024)  // a launch holds less than 2^32 threads
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence: sequences, tokens or dim too large");
    if (!cu_seqlens || !lam) return fail(NSOSX_ERR_INVALID, "gated_recurrence: null pointer");
    if (T == 0) {
        if (final_state) launch_empty(initial_state, sd, final_state, st);
        return check_launch("gated_recurrence");
    }
    if (!x || !rg || !ig || !y || !workspace)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: null pointer");
    if (T > 1 && (x_stride < D || rg_stride < D || ig_stride < D || y_stride < D))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: a row stride is less than dim");
    const int64_t size = dtype_bytes(act_dtype);
    if (views_cross(y, y_stride, x, x_stride, T, D, size) || views_cross(y, y_stride, rg, rg_stride, T, D, size) ||
        views_cross(y, y_stride, ig, ig_stride, T, D, size))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: y overlaps an input");
    if (final_state && initial_state && overlaps(final_state, sd * 4, initial_state, sd * 4))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: final_state overlaps initial_state");
    RecFwd p{x, rg, ig, x_stride, rg_stride, ig_stride, lam, rate, cu_seqlens, S, T, D, zero_rest,
             initial_state, y, y_stride, final_state, carry, static_cast<float2*>(workspace)};
    if (!carry) p.carry = reinterpret_cast<float*>(p.agg + rec_tiles(T) * D);
    if (act_dtype == NSOSX_F32) {
        if (D > 1) launch_recurrence<NSOSX_F32, 2>(p, st);
        else launch_recurrence<NSOSX_F32, 1>(p, st);
    } else {
        if (D > 1) launch_recurrence<NSOSX_BF16, 2>(p, st);
        else launch_recurrence<NSOSX_BF16, 1>(p, st);
    }
    return check_launch("gated_recurrence");
}

extern "C" int64_t nsosx_gated_recurrence_backward_workspace(int T, int D) {
    if (T <= 0 || D <= 0) return 0;
    return rec_tiles(T) * D * 16;
}

extern "C" int nsosx_gated_recurrence_backward(
    const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* rg, int64_t rg_stride,
    const void* ig, int64_t ig_stride, const float* lam, float rate, const int32_t* cu_seqlens, int S,
    int T, int D, int act_dtype, const float* initial_state, const float* carry, const float* dfinal,
    int zero_rest, void* dx, int64_t dx_stride, void* drg, int64_t drg_stride, void* dig,
    int64_t dig_stride, float* dlam, float* dinitial, void* workspace, void* stream) {
    if (const char* why = rec_check(S, T, D, act_dtype, rate))
        return fail(NSOSX_ERR_INVALID, std::string("gated_recurrence_backward: ") + why);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t sd = (int64_t)S * D;
    if (D > kRecMaxDim || sd > 0xffffffffLL - 256 || rec_tiles(T) * ((D + 63) / 64) > 0xffffffffLL / 1024)
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence_backward: sequences, tokens or dim too large");
    if (!cu_seqlens || !lam || !dlam)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: null pointer");
    if (T == 0) {
        if (dinitial) launch_empty(dfinal, sd, dinitial, st);
        launch_empty(nullptr, D, dlam, st);
        return check_launch("gated_recurrence_backward");
    }
    if (!dy || !x || !rg || !ig || !carry || !dx || !drg || !dig || !workspace)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: null pointer");
    if (T > 1 && (dy_stride < D || x_stride < D || rg_stride < D || ig_stride < D || dx_stride < D ||
                  drg_stride < D || dig_stride < D))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: a row stride is less than dim");
    const int64_t size = dtype_bytes(act_dtype);
    const void* in[4] = {dy, x, rg, ig};
    const int64_t in_s[4] = {dy_stride, x_stride, rg_stride, ig_stride};
    const void* out[3] = {dx, drg, dig};
    const int64_t out_s[3] = {dx_stride, drg_stride, dig_stride};
    for (int o = 0; o < 3; ++o) {
        for (int i = 0; i < 4; ++i)
            if (views_cross(out[o], out_s[o], in[i], in_s[i], T, D, size))
                return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: a gradient overlaps an input");
        for (int i = 0; i < o; ++i)
            if (views_cross(out[o], out_s[o], out[i], out_s[i], T, D, size))
                return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: the gradients overlap");
    }
    if (dinitial && ((dfinal && overlaps(dinitial, sd * 4, dfinal, sd * 4)) ||
                     (initial_state && overlaps(dinitial, sd * 4, initial_state, sd * 4))))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: dinitial overlaps an input");
    RecBwd p{dy, x, rg, ig, dy_stride, x_stride, rg_stride, ig_stride, lam, rate, cu_seqlens, S, T, D,
             zero_rest, initial_state, carry, dfinal, dx, drg, dig, dx_stride, drg_stride, dig_stride,
             dinitial, nullptr, static_cast<float2*>(workspace), nullptr};
    p.mcarry = reinterpret_cast<float*>(p.agg + rec_tiles(T) * D);
    p.dlam_part = p.mcarry + rec_tiles(T) * D;
    if (act_dtype == NSOSX_F32) {
        if (D > 1) launch_recurrence_bwd<NSOSX_F32, 2>(p, st);
        else launch_recurrence_bwd<NSOSX_F32, 1>(p, st);
    } else {
        if (D > 1) launch_recurrence_bwd<NSOSX_BF16, 2>(p, st);
        else launch_recurrence_bwd<NSOSX_BF16, 1>(p, st);
    }
    hipLaunchKernelGGL(recurrence_dlam_kernel, dim3((D + 63) / 64), dim3(1024), 0, st, p.dlam_part,
                       (int)rec_tiles(T), D, lam, dlam);
    return check_launch("gated_recurrence_backward");
}

extern "C" int nsosx_gated_recurrence_step(const void* x, int64_t x_stride, const void* rg,
                                           int64_t rg_stride, const void* ig, int64_t ig_stride,
                                           const float* lam, float rate, int rows, int D, int act_dtype,
                                           const float* state, float* state_out, void* y,
                                           int64_t y_stride, void* stream) {
    if (const char* why = rec_check(0, rows, D, act_dtype, rate))
        return fail(NSOSX_ERR_INVALID, std::string("gated_recurrence_step: ") + why);
    if (rows == 0) return NSOSX_OK;
    if (!x || !rg || !ig || !lam || !state || !state_out || !y)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: null pointer");
    if (rows > 1 && (x_stride < D || rg_stride < D || ig_stride < D || y_stride < D))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: a row stride is less than dim");
    const int64_t n = (int64_t)rows * D * 4, size = dtype_bytes(act_dtype);
    if (crosses(state_out, n, state, n))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: state_out may be state, but not cross it");
    if (views_cross(y, y_stride, x, x_stride, rows, D, size) ||
        views_cross(y, y_stride, rg, rg_stride, rows, D, size) ||
        views_cross(y, y_stride, ig, ig_stride, rows, D, size))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: y overlaps an input");
    const int64_t gx = (D - 1) / 256 + 1, gy = ((int64_t)rows + kStepRows - 1) / kStepRows;
    if (D > kRecMaxDim || gy > 65535 || gx * gy > 0xffffffffLL / 256)
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence_step: rows or dim too large");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)gx, (unsigned)gy);
#define NSOSX_RS(DT)                                                                                 \
    hipLaunchKernelGGL((recurrence_step_kernel<DT>), grid, dim3(256), 0, st, x, x_stride, rg, rg_stride, \
                       ig, ig_stride, lam, rate, rows, D, state, state_out, y, y_stride)
    if (act_dtype == NSOSX_F32) NSOSX_RS(NSOSX_F32);
    else NSOSX_RS(NSOSX_BF16);
#undef NSOSX_RS
    return check_launch("gated_recurrence_step");
}
