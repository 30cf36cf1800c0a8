// Gated linear recurrence over packed ragged batches, its gradients and its single-token step, on
// gfx950.  Per channel, with sr = sigmoid(rg), s = sigmoid(ig):
//   g = rate softplus(lam) sr,  a = exp(-g),  beta = sqrt(1 - a^2),  h_t = a_t h_(t-1) + beta_t s_t x_t
// The tokens of the whole batch are one stream, cut into tiles of kTile tokens whatever the sequences'
// lengths: a token that starts a sequence takes h from that sequence's initial state instead of from the
// token before it, so no tile knows or waits for the longest sequence.
// A tile's effect on what enters it is h -> A h + H, with A the product of its decays (0 where a
// sequence starts inside).  One pass: each tile's workgroup leaves its pair (A, H), finds the state that
// enters it from the pairs of the tiles before it (state_before()) and runs its tokens, still in
// registers, from there, so every input is read once.
// Backwards the same stream runs the other way in m_t = a_t dh_t, dh_t = dy_t + m_(t+1): a sequence's
// last token takes dfinal in place of m_(t+1), its first token's m is dinitial.  h is formed again
// from the forward's states at the tiles' borders (f32, one per kTile tokens), so y is not read.
#include "train.hpp"

#include <type_traits>

namespace nsosx {

constexpr int kTile = 128;      // tokens of a tile of the forward pass
constexpr int kKept = 64;       // the distance of the kept states: a tile of the gradients
constexpr int64_t kRecMaxStride = 1 << 22;  // elements: a tile's rows within 32-bit byte offsets
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// A tile's rows of a [T, D] view: base, a lane's byte offset in a row, the row's byte offset in a scalar
// register (always of a real row: nothing here leans on the resource's range check).
struct Rows {
    __amdgpu_buffer_rsrc_t r;
    uint32_t row;  // bytes
};

template <int DT>
__device__ __forceinline__ Rows tile_rows(const void* p, int64_t stride, int64_t t0) {
    constexpr int size = DT == NSOSX_F32 ? 4 : 2;
    return {make_rsrc(static_cast<const char*>(p) + t0 * stride * size, 0xffffffffu), (uint32_t)(stride * size)};
}

// Two neighbouring channels of a token (one where D is 1), as loaded, at any alignment.
template <int DT, int V> struct Pair;
template <> struct Pair<NSOSX_BF16, 2> {
    uint32_t w;
    __device__ __forceinline__ void load(const Rows& v, uint32_t lane, int row) {
        w = __builtin_amdgcn_raw_buffer_load_b32(v.r, lane, row * v.row, 0);
    }
    __device__ __forceinline__ float get(int k) const {
        return __uint_as_float(k ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ void store(const Rows& v, uint32_t lane, int row, const float (&f)[2]) {
        __builtin_amdgcn_raw_buffer_store_b32(pack_bf16x2(f[0], f[1]), v.r, lane, row * v.row, 0);
    }
};
template <> struct Pair<NSOSX_F32, 2> {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 w;
    __device__ __forceinline__ void load(const Rows& v, uint32_t lane, int row) {
        w = __builtin_amdgcn_raw_buffer_load_b64(v.r, lane, row * v.row, 0);
    }
    __device__ __forceinline__ float get(int k) const { return __uint_as_float(k ? w.y : w.x); }
    static __device__ __forceinline__ void store(const Rows& v, uint32_t lane, int row, const float (&f)[2]) {
        const u32x2 w = {__float_as_uint(f[0]), __float_as_uint(f[1])};
        __builtin_amdgcn_raw_buffer_store_b64(w, v.r, lane, row * v.row, 0);
    }
};
template <int DT> struct Pair<DT, 1> {
    float v;
    __device__ __forceinline__ void load(const Rows& p, uint32_t lane, int row) {
        v = raw_to_f32<DT>(buf_load_raw<DT>(p.r, lane + row * p.row));
    }
    __device__ __forceinline__ float get(int) const { return v; }
    static __device__ __forceinline__ void store(const Rows& p, uint32_t lane, int row, const float (&f)[1]) {
        buf_store_act<DT>(p.r, lane + row * p.row, f[0]);
    }
};

// e^-x and 1 / (1 + e^-x) on the exponential and reciprocal units; the latter is off by up to
// (5 + 2 |x|) half steps.
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * -kLog2e); }
__device__ __forceinline__ float sigmoid_of(float e) { return __builtin_amdgcn_rcpf(1.0f + e); }

// 1 - sigmoid = e^-x sigmoid, without the cancellation of large x.  Where e^-x has overflowed and the
// sigmoid is 0 it reads 0: what it multiplies holds the sigmoid too.
__device__ __forceinline__ float rest_of(float e, float s) {
    return __builtin_amdgcn_fmed3f(e, 0.0f, 3.0e38f) * s;
}

// rate softplus(lam) in units of log 2: a = 2^(-k2 sr)
__device__ __forceinline__ float decay_rate(float lam, float rate) {
    return rate * (fmaxf(lam, 0.0f) + log1pf(expf(-fabsf(lam)))) * kLog2e;
}

// p = 1 - a^2 for a = 2^-q.  Where a is near 1 the difference would cancel: below t = -log(a^2) = 0.25
// (q = kSmall) it is q times a fit of (1 - e^-t) / t in q (own least-squares fit, relative error 1e-7 with
// its roundings); above, 1 - a^2 is exact to 7e-7.
constexpr float kSmall = 0.18033688f;

__device__ __forceinline__ float one_less_square_small(float q) {
    float f = __fmaf_rn(q, 0.038452983f, -0.1532337f);
    f = __fmaf_rn(q, f, 0.44399065f);
    f = __fmaf_rn(q, f, -0.9609051f);
    f = __fmaf_rn(q, f, 1.3862944f);
    return q * f;
}

template <bool SMALL>
__device__ __forceinline__ float one_less_square(float q, float a) {
    const float p = one_less_square_small(q);
    return SMALL || q < kSmall ? p : __fmaf_rn(-a, a, 1.0f);
}

// Where the tile's sequences start and end: s_start[i] / s_end[i] hold the sequence whose first /
// last token is token i of the tile, else -1.  Every workgroup reads all of cu_seqlens, a few loads
// that do not depend on each other, rather than search it in log2(S) that do.
template <int NT, int L>
__device__ __forceinline__ void tile_borders(const int32_t* __restrict__ cu, int S, int64_t t0,
                                             int32_t* s_start, int32_t* s_end) {
    for (int i = threadIdx.x; i < L; i += NT) s_start[i] = s_end[i] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < S; s += NT) {
        const int64_t lo = cu[s], hi = cu[s + 1];
        if (hi <= lo) continue;
        if (lo >= t0 && lo < t0 + L) s_start[lo - t0] = s;
        if (hi > t0 && hi <= t0 + L) s_end[hi - 1 - t0] = s;
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
    const bool mine = lane < R;
    starts = (uint32_t)__ballot(mine & (s_start[i] >= 0));
    ends = (uint32_t)__ballot(mine & (s_end[i] >= 0));
    inside = (uint32_t)__ballot(mine & (t >= lo) & (t < hi));
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

// ---- the state that enters a tile ---------------------------------------------------
//
// A word per (tile, channel) in the order of the scan: 0 until the tile has something to say, then its
// pair (A's bits with the sign set, H), then the state behind it (kWhole, P).  Words are 64 bits, written
// and read whole at device scope, so nothing else needs to be ordered with them.
// P_k = fma(A_k, P_(k-1), H_k) always, however far back a tile finds a P: the same bits every run.
// Every wait ends: workgroups take their tiles by a ticket, in the order of the scan, so whoever waits
// waits for workgroups that have started, and those leave their pair before they wait themselves.
constexpr uint32_t kWhole = 1;
constexpr int kWindow = 4;          // tiles looked back at a time
constexpr int kMaxPolls = 1 << 22;  // seconds; then the state is NaN and the kernel ends

__device__ __forceinline__ void leave(uint64_t* word, uint32_t tag, float v) {
    __hip_atomic_store(word, ((uint64_t)tag << 32) | __float_as_uint(v), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

// One wave, V channels a lane: tile k of the scan has the pair (A, H); c becomes the state before it.
template <int V>
__device__ __forceinline__ void state_before(uint64_t* words, int64_t k, int64_t D, uint32_t ch,
                                             const float (&A)[V], const float (&H)[V], float (&c)[V]) {
    uint64_t* mine = words + k * D + ch;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        // nothing enters the first tile, and nothing passes a sequence's border
        const bool whole = k == 0 || A[v] == 0.0f;
        leave(mine + v, whole ? kWhole : __float_as_uint(A[v]) | 0x80000000u, H[v]);
        c[v] = 0.0f;
    }
    if (k == 0) return;
    bool done = false;
    for (int polls = 0; !__all(done); ++polls) {
        if (polls > 0) __builtin_amdgcn_s_sleep(1);
        uint64_t w[kWindow][V];
#pragma unroll
        for (int i = 0; i < kWindow; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v)
                w[i][v] = __hip_atomic_load(words + max(k - 1 - i, (int64_t)0) * D + (ch + v), __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
        done = true;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            int found = kWindow;  // the nearest tile whose P is known, behind nothing but pairs
#pragma unroll
            for (int i = kWindow - 1; i >= 0; --i) {
                const uint32_t tag = (uint32_t)(w[i][v] >> 32);
                found = tag == kWhole ? i : tag == 0 ? kWindow : found;
            }
            float s = 0.0f;
#pragma unroll
            for (int i = kWindow - 1; i >= 0; --i) {
                const float a = __uint_as_float((uint32_t)(w[i][v] >> 32) & 0x7fffffffu);
                const float h = __uint_as_float((uint32_t)w[i][v]);
                s = i == found ? h : i < found ? __fmaf_rn(a, s, h) : s;
            }
            c[v] = s;
            done = done && found < kWindow;
        }
        if (polls >= kMaxPolls) {
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = __builtin_nanf("");
            break;
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (A[v] != 0.0f) leave(mine + v, kWhole, __fmaf_rn(A[v], c[v], H[v]));
}

// The workgroup's place in the scan: ticket, or its index where there is one tile in time.
__device__ __forceinline__ int take_ticket(uint32_t* ticket) {
    if (!ticket) return blockIdx.x;
    __shared__ uint32_t s_ticket;
    if (threadIdx.x == 0) s_ticket = atomicAdd(ticket, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(s_ticket);
}

__global__ __launch_bounds__(256) void recurrence_clear_kernel(uint4* __restrict__ p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}

// A state row a sequence brings in, or zeros.
template <int V>
__device__ __forceinline__ void take_state(const float* from, int s, int D, int ch, float (&h)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = from ? from[(int64_t)s * D + ch + k] : 0.0f;
}

template <int V>
__device__ __forceinline__ void put_state(float* to, int s, int D, int ch, const float (&h)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) to[(int64_t)s * D + ch + k] = h[k];
}

// h -> A h + H; A = 0 passes nothing on, whatever h holds (it may be another sequence's infinity)
__device__ __forceinline__ float through(float A, float H, float h) {
    return A == 0.0f ? H : __fmaf_rn(A, h, H);
}

// What a workgroup and a wave of it work on.
struct Place {
    int64_t t0, order;              // first token; the tile's number in the scan
    int ch, cb, lane, wave, real;   // the lane's first channel, the block's; tokens the tile really has
    bool act;                       // false: a lane past the last channel, which computes the last ones again
    uint32_t starts, ends, inside;  // a bit per token of the wave
};

template <int V, int L, int R>
__device__ __forceinline__ Place find_place(uint32_t* ticket, int T, int D, bool reverse) {
    Place p;
    p.lane = threadIdx.x & 63;
    p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (D - 1) / (64 * V) + 1, at = take_ticket(ticket), order = at / blocks;
    const int c0 = (at - order * blocks) * 64 * V;
    p.order = order;
    p.t0 = (int64_t)(reverse ? (T - 1) / L - order : order) * L;
    p.ch = min(c0 + p.lane * V, D - V);
    p.cb = min(c0, D - V);
    p.act = c0 + p.lane * V < D;
    p.real = (int)min((int64_t)L, T - p.t0);
    return p;
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
    float *final, *carry;  // carry [T / kKept up, D]: the state before every kKept-th token
    uint32_t* ticket;      // NULL where there is one tile in time
    uint64_t* words;       // [tiles, D]
};

// A workgroup takes a tile of 128 channels, two a lane; each wave takes R of the tile's tokens.
template <int DT, int V, int R>
__global__ __launch_bounds__(64 * (kTile / R), 4) void recurrence_kernel(RecFwd P) {
    constexpr int L = kTile, WAVES = L / R, NT = 64 * WAVES;
    constexpr uint32_t ALL = (1u << R) - 1;
    __shared__ int32_t s_start[L], s_end[L];
    __shared__ float s_k2[64 * V], s_c[V][64], s_a[WAVES][V][64], s_h[WAVES][V][64];
    Place p = find_place<V, L, R>(P.ticket, P.T, P.D, false);
    const int lane = p.lane, wave = p.wave, ch = p.ch;
    const uint32_t off = ch * (DT == NSOSX_F32 ? 4 : 2);
    float a[R][V], u[R][V];
    {
        Pair<DT, V> x[R], r[R], g[R];
        const Rows vx = tile_rows<DT>(P.x, P.xs, p.t0), vr = tile_rows<DT>(P.rg, P.rs, p.t0),
                   vg = tile_rows<DT>(P.ig, P.is, p.t0);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int t = min(wave * R + j, p.real - 1);
            r[j].load(vr, off, t);
            g[j].load(vg, off, t);
            x[j].load(vx, off, t);
        }
        for (int i = threadIdx.x; i < 64 * V; i += NT)
            s_k2[i] = decay_rate(P.lam[min(p.cb + i, P.D - 1)], P.rate);
        tile_borders<NT, L>(P.cu, P.S, p.t0, s_start, s_end);
        wave_masks<R>(s_start, s_end, wave, p.t0, P.cu[0], min(P.cu[P.S], P.T), p.starts, p.ends, p.inside);
        float k2[V];
        bool small = true;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            k2[k] = s_k2[ch - p.cb + k];
            small = small && k2[k] < kSmall;
        }
        auto gates = [&](auto fits) {
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float q = k2[k] * sigmoid_of(exp_neg(r[j].get(k)));
                    a[j][k] = __builtin_amdgcn_exp2f(-q);
                    u[j][k] = __builtin_amdgcn_sqrtf(one_less_square<decltype(fits)::value>(q, a[j][k])) *
                              (sigmoid_of(exp_neg(g[j].get(k))) * x[j].get(k));
                }
        };
        // (decays that stay above 0.88 even at open gates, as most do, take a third fewer steps)
        if (__all(small)) gates(std::true_type{});
        else gates(std::false_type{});
    }
    const bool plain = !p.starts && !p.ends && p.inside == ALL;  // no border, no row of no sequence
    float A[V], H[V];
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
    auto local = [&](auto borders) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool start = decltype(borders)::value && (p.starts >> j & 1);
            if (start) take_state<V>(P.initial, s_start[wave * R + j], P.D, ch, H);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
                A[k] = start ? 0.0f : A[k] * a[j][k];
            }
        }
    };
    if (plain) local(std::false_type{});
    else local(std::true_type{});
#pragma unroll
    for (int k = 0; k < V; ++k) s_a[wave][k][lane] = A[k], s_h[wave][k][lane] = H[k];
    __syncthreads();
    if (wave == 0) {
        float c[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            c[k] = 0.0f;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                const float aw = s_a[w][k][lane];
                H[k] = through(aw, s_h[w][k][lane], H[k]);
                A[k] = aw == 0.0f ? 0.0f : A[k] * aw;
            }
        }
        if (P.ticket) state_before<V>(P.words, p.order, P.D, ch, A, H, c);
#pragma unroll
        for (int k = 0; k < V; ++k) s_c[k][lane] = c[k];
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        h[k] = s_c[k][lane];
        for (int w = 0; w < wave; ++w) h[k] = through(s_a[w][k][lane], s_h[w][k][lane], h[k]);
    }
    if (wave * R % kKept == 0 && P.carry && wave * R < p.real && p.act)
        put_state<V>(P.carry, (int)((p.t0 + wave * R) / kKept), P.D, ch, h);
    const Rows vy = tile_rows<DT>(P.y, P.ys, p.t0);
    auto apply = [&](auto borders) {
        constexpr bool B = decltype(borders)::value;
        const float zero[V] = {};
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int t = wave * R + j;
            if (B && !(p.inside >> j & 1)) {
                if (P.rest && t < p.real && p.act) Pair<DT, V>::store(vy, off, t, zero);
                continue;
            }
            if (B && (p.starts >> j & 1)) take_state<V>(P.initial, s_start[t], P.D, ch, h);
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = __fmaf_rn(a[j][k], h[k], u[j][k]);
            if (p.act) Pair<DT, V>::store(vy, off, t, h);
            if (B && (p.ends >> j & 1) && P.final && p.act) put_state<V>(P.final, s_end[t], P.D, ch, h);
        }
    };
    if (plain) apply(std::false_type{});
    else apply(std::true_type{});
    if (p.order == 0 && P.final) empty_states<V, NT>(P.cu, P.S, P.D, ch, p.act, P.initial, P.final);
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
    uint32_t* ticket;
    uint64_t* words;  // [tiles, D], of the reversed stream
};

// The same from the last tile to the first.  With q = g / log 2, w = a q and b2 = p = 1 - a^2:
//   e = dh (s x a w / beta - w h_before), in units of log 2;  what 1 / beta multiplies goes to 0 with it
template <int DT, int V, int R>
__global__ __launch_bounds__(64 * (kKept / R), 4) void recurrence_bwd_kernel(RecBwd P) {
    constexpr int L = kKept, WAVES = L / R, NT = 64 * WAVES;
    constexpr uint32_t ALL = (1u << R) - 1;
    __shared__ int32_t s_start[L], s_end[L];
    __shared__ float s_k2[64 * V], s_c[V][64], s_a[WAVES][V][64], s_h[WAVES][V][64], s_b[WAVES][V][64],
        s_m[WAVES][V][64];
    Place p = find_place<V, L, R>(P.ticket, P.T, P.D, true);
    const int lane = p.lane, wave = p.wave, ch = p.ch;
    const uint32_t off = ch * (DT == NSOSX_F32 ? 4 : 2);
    // kept over the wait: a, u (then the state before each token), e^-rg, e^-ig, x and dy as loaded
    float a[R][V], u[R][V], er[R][V], eg[R][V], k2[V];
    Pair<DT, V> x[R], d[R];
    float h0[V];
    {
        Pair<DT, V> r[R], g[R];
        const Rows vx = tile_rows<DT>(P.x, P.xs, p.t0), vr = tile_rows<DT>(P.rg, P.rs, p.t0),
                   vg = tile_rows<DT>(P.ig, P.is, p.t0), vd = tile_rows<DT>(P.dy, P.dys, p.t0);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int t = min(wave * R + j, p.real - 1);
            r[j].load(vr, off, t);
            g[j].load(vg, off, t);
            x[j].load(vx, off, t);
            d[j].load(vd, off, t);
        }
        take_state<V>(P.carry, (int)(p.t0 / kKept), P.D, ch, h0);
        for (int i = threadIdx.x; i < 64 * V; i += NT)
            s_k2[i] = decay_rate(P.lam[min(p.cb + i, P.D - 1)], P.rate);
        tile_borders<NT, L>(P.cu, P.S, p.t0, s_start, s_end);
        wave_masks<R>(s_start, s_end, wave, p.t0, P.cu[0], min(P.cu[P.S], P.T), p.starts, p.ends, p.inside);
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                er[j][k] = exp_neg(r[j].get(k));
                eg[j][k] = exp_neg(g[j].get(k));
            }
    }
    bool small = true;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        k2[k] = s_k2[ch - p.cb + k];
        small = small && k2[k] < kSmall;
    }
    small = __all(small);
    auto gates = [&](auto fits) {
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float q = k2[k] * sigmoid_of(er[j][k]);
                a[j][k] = __builtin_amdgcn_exp2f(-q);
                u[j][k] = __builtin_amdgcn_sqrtf(one_less_square<decltype(fits)::value>(q, a[j][k])) *
                          (sigmoid_of(eg[j][k]) * x[j].get(k));
            }
    };
    if (small) gates(std::true_type{});
    else gates(std::false_type{});
    const bool plain = !p.starts && !p.ends && p.inside == ALL;
    float A[V], H[V], B[V], M[V];
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = B[k] = 1.0f, H[k] = M[k] = 0.0f;
    auto local = [&](auto borders) {
        constexpr bool BORDERS = decltype(borders)::value;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool start = BORDERS && (p.starts >> j & 1);
            if (start) take_state<V>(P.initial, s_start[wave * R + j], P.D, ch, H);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
                A[k] = start ? 0.0f : A[k] * a[j][k];
            }
        }
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            const bool end = BORDERS && (p.ends >> j & 1), out = BORDERS && !(p.inside >> j & 1);
            if (end) take_state<V>(P.dfinal, s_end[wave * R + j], P.D, ch, M);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                M[k] = out ? 0.0f : a[j][k] * (d[j].get(k) + M[k]);
                B[k] = end || out ? 0.0f : B[k] * a[j][k];
            }
        }
    };
    if (plain) local(std::false_type{});
    else local(std::true_type{});
#pragma unroll
    for (int k = 0; k < V; ++k) {
        s_a[wave][k][lane] = A[k], s_h[wave][k][lane] = H[k];
        s_b[wave][k][lane] = B[k], s_m[wave][k][lane] = M[k];
    }
    __syncthreads();
    if (wave == WAVES - 1) {
        float c[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            c[k] = 0.0f;
#pragma unroll
            for (int w = WAVES - 2; w >= 0; --w) {
                const float bw = s_b[w][k][lane];
                M[k] = through(bw, s_m[w][k][lane], M[k]);
                B[k] = bw == 0.0f ? 0.0f : B[k] * bw;
            }
        }
        if (P.ticket) state_before<V>(P.words, p.order, P.D, ch, B, M, c);
#pragma unroll
        for (int k = 0; k < V; ++k) s_c[k][lane] = c[k];
    }
    float h[V], m[V], e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        h[k] = h0[k];
        for (int w = 0; w < wave; ++w) h[k] = through(s_a[w][k][lane], s_h[w][k][lane], h[k]);
    }
    // u becomes the state before each token
    auto states = [&](auto borders) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (decltype(borders)::value && (p.starts >> j & 1))
                take_state<V>(P.initial, s_start[wave * R + j], P.D, ch, h);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float before = h[k];
                h[k] = __fmaf_rn(a[j][k], h[k], u[j][k]);
                u[j][k] = before;
            }
        }
    };
    if (plain) states(std::false_type{});
    else states(std::true_type{});
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) {
        m[k] = s_c[k][lane];
        for (int w = WAVES - 1; w > wave; --w) m[k] = through(s_b[w][k][lane], s_m[w][k][lane], m[k]);
        e[k] = 0.0f;
    }
    // (the compiler would keep the gates since their first use, in registers that are not there)
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) asm volatile("" : "+v"(er[j][k]), "+v"(eg[j][k]));
    const Rows vx = tile_rows<DT>(P.dx, P.dxs, p.t0), vr = tile_rows<DT>(P.drg, P.drs, p.t0),
               vg = tile_rows<DT>(P.dig, P.dis, p.t0);
    auto apply = [&](auto borders, auto fits) {
        constexpr bool BORDERS = decltype(borders)::value;
        const float zero[V] = {};
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            const int t = wave * R + j;
            if (BORDERS && !(p.inside >> j & 1)) {
                if (P.rest && t < p.real && p.act) {
                    Pair<DT, V>::store(vx, off, t, zero);
                    Pair<DT, V>::store(vr, off, t, zero);
                    Pair<DT, V>::store(vg, off, t, zero);
                }
                continue;
            }
            if (BORDERS && (p.ends >> j & 1)) take_state<V>(P.dfinal, s_end[t], P.D, ch, m);
            float ox[V], orr[V], oi[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float sr = sigmoid_of(er[j][k]), si = sigmoid_of(eg[j][k]);
                const float q = k2[k] * sr, xv = x[j].get(k), av = a[j][k];
                const float b2 = one_less_square<decltype(fits)::value>(q, av);
                const float rb = __builtin_amdgcn_rsqf(fmaxf(b2, 1e-37f));  // 1 / beta
                const float w = av * q, dh = d[j].get(k) + m[k];
                const float ev = dh * __fmaf_rn(si * xv, av * w * rb, -(w * u[j][k]));
                ox[k] = dh * (b2 * rb) * si;
                oi[k] = ox[k] * xv * rest_of(eg[j][k], si);
                orr[k] = ev * rest_of(er[j][k], sr) * kLn2;
                e[k] += ev;
                m[k] = av * dh;
            }
            if (p.act) {
                Pair<DT, V>::store(vx, off, t, ox);
                Pair<DT, V>::store(vr, off, t, orr);
                Pair<DT, V>::store(vg, off, t, oi);
            }
            if (BORDERS && (p.starts >> j & 1) && P.dinitial && p.act)
                put_state<V>(P.dinitial, s_start[t], P.D, ch, m);
        }
    };
    if (!plain) apply(std::true_type{}, std::false_type{});
    else if (small) apply(std::false_type{}, std::true_type{});
    else apply(std::false_type{}, std::false_type{});
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) s_a[wave][k][lane] = e[k];
    __syncthreads();
    if (wave == 0 && p.act) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            for (int w = 1; w < WAVES; ++w) e[k] += s_a[w][k][lane];
        put_state<V>(P.dlam_part, (int)(p.t0 / L), P.D, ch, e);
    }
    if (p.order == 0 && P.dinitial) empty_states<V, NT>(P.cu, P.S, P.D, ch, p.act, P.dfinal, P.dinitial);
}

// dlam = sigmoid(lam) / softplus(lam) * sum_t e, e in units of log 2: the tiles' sums in a fixed order (64 channels a
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
    dlam[c] = sum * kLn2 * (sp == 0.0f ? 1.0f : sig / sp);
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
        const float q = k2 * sigmoid_of(exp_neg(load_act<DT>(rg, r * rs + c))), a = __builtin_amdgcn_exp2f(-q);
        const float u = __builtin_amdgcn_sqrtf(one_less_square<false>(q, a)) *
                        (sigmoid_of(exp_neg(load_act<DT>(ig, r * is + c))) * load_act<DT>(x, r * xs + c));
        const float h = __fmaf_rn(a, state[r * D + c], u);
        state_out[r * D + c] = h;
        store_act<DT>(y, r * ys + c, h);
    }
}

static int64_t rec_tiles(int64_t T, int tile) { return (T + tile - 1) / tile; }

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

// ticket (16 bytes), then the words
static int64_t rec_words_bytes(int64_t tiles, int D) { return tiles > 1 ? 16 + (tiles * D * 8 + 15) / 16 * 16 : 0; }

template <typename P>
static void clear_words(P& p, int64_t tiles, void* workspace, hipStream_t st) {
    p.ticket = nullptr;
    p.words = nullptr;
    if (tiles == 1) return;
    const int64_t n = rec_words_bytes(tiles, p.D) / 16;
    p.ticket = static_cast<uint32_t*>(workspace);
    p.words = reinterpret_cast<uint64_t*>(p.ticket + 4);
    hipLaunchKernelGGL(recurrence_clear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st,
                       static_cast<uint4*>(workspace), n);
}

template <int DT, int V>
static void launch_recurrence(const RecFwd& p, hipStream_t st) {
    const dim3 grid((unsigned)(rec_tiles(p.T, kTile) * ((p.D - 1) / (64 * V) + 1)));
    hipLaunchKernelGGL((recurrence_kernel<DT, V, 16>), grid, dim3(64 * (kTile / 16)), 0, st, p);
}

template <int DT, int V>
static void launch_recurrence_bwd(const RecBwd& p, hipStream_t st) {
    const dim3 grid((unsigned)(rec_tiles(p.T, kKept) * ((p.D - 1) / (64 * V) + 1)));
    hipLaunchKernelGGL((recurrence_bwd_kernel<DT, V, 8>), grid, dim3(64 * (kKept / 8)), 0, st, p);
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

extern "C" int nsosx_gated_recurrence_tile(void) { return kKept; }

extern "C" int64_t nsosx_gated_recurrence_workspace(int T, int D) {
    if (T <= 0 || D <= 0) return 0;
    return rec_words_bytes(rec_tiles(T, kTile), D);
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
    if (D > kRecMaxStride || sd > 0xffffffffLL - 256 ||
        rec_tiles(T, kTile) * ((D + 63) / 64) > 0xffffffffLL / 1024)  // a launch holds less than 2^32 threads
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence: sequences, tokens or dim too large");
    if (!cu_seqlens || !lam) return fail(NSOSX_ERR_INVALID, "gated_recurrence: null pointer");
    if (T == 0) {
        if (final_state) launch_empty(initial_state, sd, final_state, st);
        return check_launch("gated_recurrence");
    }
    if (!x || !rg || !ig || !y || (!workspace && rec_tiles(T, kTile) > 1))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: null pointer");
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: workspace must be 16-byte aligned");
    if (T > 1 && (x_stride < D || rg_stride < D || ig_stride < D || y_stride < D))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: a row stride is less than dim");
    if (T > 1 && (x_stride > kRecMaxStride || rg_stride > kRecMaxStride || ig_stride > kRecMaxStride ||
                  y_stride > kRecMaxStride))
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence: a row stride is more than 2^22");
    const int64_t size = dtype_bytes(act_dtype);
    if (views_cross(y, y_stride, x, x_stride, T, D, size) || views_cross(y, y_stride, rg, rg_stride, T, D, size) ||
        views_cross(y, y_stride, ig, ig_stride, T, D, size))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: y overlaps an input");
    if (final_state && initial_state && overlaps(final_state, sd * 4, initial_state, sd * 4))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: final_state overlaps initial_state");
    RecFwd p{x, rg, ig, x_stride, rg_stride, ig_stride, lam, rate, cu_seqlens, S, T, D, zero_rest,
             initial_state, y, y_stride, final_state, carry, nullptr, nullptr};
    clear_words(p, rec_tiles(T, kTile), workspace, st);
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
    return rec_words_bytes(rec_tiles(T, kKept), D) + rec_tiles(T, kKept) * D * 4;
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
    if (D > kRecMaxStride || sd > 0xffffffffLL - 256 || rec_tiles(T, kKept) * ((D + 63) / 64) > 0xffffffffLL / 1024)
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
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: workspace must be 16-byte aligned");
    if (T > 1 && (dy_stride < D || x_stride < D || rg_stride < D || ig_stride < D || dx_stride < D ||
                  drg_stride < D || dig_stride < D))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_backward: a row stride is less than dim");
    if (T > 1 && (dy_stride > kRecMaxStride || x_stride > kRecMaxStride || rg_stride > kRecMaxStride ||
                  ig_stride > kRecMaxStride || dx_stride > kRecMaxStride || drg_stride > kRecMaxStride ||
                  dig_stride > kRecMaxStride))
        return fail(NSOSX_ERR_OVERFLOW, "gated_recurrence_backward: a row stride is more than 2^22");
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
             dinitial, reinterpret_cast<float*>(static_cast<char*>(workspace) + rec_words_bytes(rec_tiles(T, kKept), D)),
             nullptr, nullptr};
    clear_words(p, rec_tiles(T, kKept), workspace, st);
    if (act_dtype == NSOSX_F32) {
        if (D > 1) launch_recurrence_bwd<NSOSX_F32, 2>(p, st);
        else launch_recurrence_bwd<NSOSX_F32, 1>(p, st);
    } else {
        if (D > 1) launch_recurrence_bwd<NSOSX_BF16, 2>(p, st);
        else launch_recurrence_bwd<NSOSX_BF16, 1>(p, st);
    }
    hipLaunchKernelGGL(recurrence_dlam_kernel, dim3((D + 63) / 64), dim3(1024), 0, st, p.dlam_part,
                       (int)rec_tiles(T, kKept), D, lam, dlam);
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
    if (D > kRecMaxStride || gy > 65535 || gx * gy > 0xffffffffLL / 256)
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
