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
// from the forward's states before every kKept-th token (f32), so y is not read.
#include "train.hpp"

#include <atomic>
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
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w)); }
    __device__ __forceinline__ float get(int k) const {
        return __uint_as_float(k ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ void store(const Rows& v, uint32_t lane, int row, const float (&f)[2]) {
        __builtin_amdgcn_raw_buffer_store_b32(pack_bf16x2(f[0], f[1]), v.r, lane, row * v.row, 0);
    }
};
template <int DT> struct Pair<DT, 1> {
    float v;
    __device__ __forceinline__ void load(const Rows& p, uint32_t lane, int row) {
        v = raw_to_f32<DT>(buf_load_raw<DT>(p.r, lane + row * p.row));
    }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(v)); }
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

// What a wave's R tokens are, a bit per token; their sequences are left in LDS.
struct Tokens {
    uint32_t starts, ends, inside;
    template <int R> __device__ __forceinline__ bool plain() const {
        return !starts && !ends && inside == (1u << R) - 1;
    }
};

// cu holds S + 1 bounds: a search per lane, in LDS but for thousands of sequences.  seqs: the wave's R.
template <int R, typename Bounds>
__device__ __forceinline__ Tokens find_tokens(const Bounds& cu, int S, int lane, int64_t first, int64_t T,
                                              int32_t* seqs) {
    const int i = min(lane, R - 1);
    const int64_t t = first + i;
    int lo = 0, hi = S + 1;  // the first bound past t: the last of several empty sequences is not t's
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    const int s = min(max(lo - 1, 0), max(S - 1, 0));
    const bool in = (lo > 0) & (lo <= S) & (t < T) & (lane < R);
    seqs[i] = s;
    Tokens r;
    r.inside = (uint32_t)__ballot(in);
    r.starts = (uint32_t)__ballot(in & (cu[s] == t));
    r.ends = (uint32_t)__ballot(in & (cu[min(s + 1, S)] == t + 1));
    return r;
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

// The product of decays, and never 0 but for a border, however strong they are: what is not finite goes on to
// the end of its sequence.  The least is 2^-149: products below 2^-126 keep the bits that they can, and of a
// finite state its 2^-149th part, 5e-7 at most, is what goes on too far.
constexpr float kLeast = 1.40129846e-45f;

__device__ __forceinline__ float joined(float A, float a) {
    return A == 0.0f || a == 0.0f ? 0.0f : fmaxf(A * a, kLeast);
}

// h -> A h + H; A = 0 passes nothing on, whatever h holds (it may be another sequence's infinity)
__device__ __forceinline__ float through(float A, float H, float h) {
    return A == 0.0f ? H : __fmaf_rn(A, h, H);
}

// ---- the state that enters a tile ---------------------------------------------------
//
// Tiles meet through words in memory, one per (tile, channel) with the tile's pair, and one per
// (group of kGroup tiles, channel) with the group's pair and later the state P behind it.  A word is 64
// bits, written and read whole at device scope, so nothing else has to be ordered with it: 0 until
// there is something to say, (A's bits with the sign set, H) for a pair, (kWhole, P) for a state.
//   P_g = A_g P_(g-1) + H_g,  a tile's state is P_(g-1) through the pairs of its group's tiles before it
// in that order however far back a group finds a P, so the bits are the same every run.
// A tile waits on flags (per 64 channels; 1: a pair is there, 2: a state), a few bytes a look, and reads
// words only when the flags say that they are there: words polled by themselves took as much time as
// everything else.  The flags are hints, the words' own tags decide.
// Every wait ends: workgroups take their tiles by a ticket, in the order of the scan, and leave a tile's
// pair before they wait for another's, so whoever waits waits for tiles that a started workgroup has
// left or will leave without waiting for a later one.  One that has looked kLooks times all the same
// gives up: it takes what it has not seen for NaN, also in the words that it leaves, so what a later tile
// makes of them is right or NaN.
constexpr uint32_t kWhole = 1;
constexpr int kGroup = 4;        // tiles
constexpr int kLooks = 1 << 22;  // seconds
constexpr uint64_t kLost = 0xbf8000007fc00000ull;  // the pair (1, NaN)

struct RecShared {
    uint32_t* ticket;           // NULL where there is one tile in time: no tile waits for another
    uint64_t *words, *groups;   // [tiles, D], [groups, D]
    uint32_t *flags, *gflags;   // [D / 64 up, tiles], [D / 64 up, groups]
    float* k2;                  // [D]: the channels' decay rates, formed once
    int spent;                  // looks that a tile starts with (kLooks: it waits for nothing)
};

__device__ __forceinline__ void leave(uint64_t* word, uint32_t tag, float v) {
    __hip_atomic_store(word, ((uint64_t)tag << 32) | __float_as_uint(v), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t look(const uint64_t* row, uint32_t bytes) {
    return __hip_atomic_load(reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(row) + bytes),
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void raise_flag(uint32_t* flag, uint32_t v) {
    if ((threadIdx.x & 63) == 0) __hip_atomic_store(flag, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint32_t see_flag(const uint32_t* flag) {
    return __hip_atomic_load(flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint32_t tag_of(uint64_t w) { return (uint32_t)(w >> 32); }
__device__ __forceinline__ float pair_a(uint64_t w) { return __uint_as_float(tag_of(w) & 0x7fffffffu); }
__device__ __forceinline__ float pair_h(uint64_t w) { return __uint_as_float((uint32_t)w); }

// One wave, a channel a lane: tile k of the scan has the pair (A, H); the return value is the state
// before it.  part: the wave's 64 channels among all; s_w [kGroup - 1] words of LDS a lane, `step` apart
// (registers are the tile's).
template <typename Shared>
__device__ __forceinline__ float state_before(const Shared& sh, int k, int tiles, int64_t D, int part, uint32_t ch,
                                              float A, float H, uint64_t* s_w, int step) {
    const int g = k / kGroup, pos = k % kGroup, lane = threadIdx.x & 63;
    const int ngroups = (tiles - 1) / kGroup + 1;
    uint32_t* flags = sh.flags + (int64_t)part * tiles;
    uint32_t* gflags = sh.gflags + (int64_t)part * ngroups;
    uint64_t* behind = sh.groups + g * D + ch;
    leave(sh.words + k * D + ch, __float_as_uint(A) | 0x80000000u, H);
    raise_flag(flags + k, 1);
    int polls = sh.spent;
    if (pos > 0) {  // the pairs of the tiles before this one in its group
        const uint64_t* row = sh.words + (int64_t)g * kGroup * D;
#pragma unroll 1
        for (bool all = false; !all && polls <= kLooks;) {
            while (!__all(see_flag(flags + g * kGroup + min(lane, pos - 1)) != 0) && ++polls <= kLooks)
                __builtin_amdgcn_s_sleep(4);
            uint64_t w[kGroup - 1];
            uint32_t at = ch * 8;
            asm volatile("" : "+v"(at));  // (or every word's address would be kept in registers)
#pragma unroll
            for (int i = 0; i < kGroup - 1; ++i)
                if (i < pos) w[i] = look(row + i * D, at);
            all = true;
#pragma unroll
            for (int i = 0; i < kGroup - 1; ++i)
                if (i < pos) {
                    all = all & (tag_of(w[i]) != 0);
                    s_w[i * step] = tag_of(w[i]) != 0 ? w[i] : kLost;
                }
            all = __all(all);
            ++polls;
        }
    }
    float Ag = 1.0f, Hg = 0.0f, c = 0.0f;
    if (pos == kGroup - 1) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            const float a = i < kGroup - 1 ? pair_a(s_w[i * step]) : A;
            Hg = through(a, i < kGroup - 1 ? pair_h(s_w[i * step]) : H, Hg);
            Ag = joined(Ag, a);
        }
        // nothing enters the first group, and nothing passes a sequence's border
        const bool whole = g == 0 || Ag == 0.0f;
        leave(behind, whole ? kWhole : __float_as_uint(Ag) | 0x80000000u, Hg);
        raise_flag(gflags + g, __all(whole) ? 2 : 1);
    }
    if (g > 0) {
        bool all = false;
#pragma unroll 1
        while (!all && polls <= kLooks) {
            int far;  // the nearest group whose state is known, with pairs of all groups between
            for (;; __builtin_amdgcn_s_sleep(4)) {
                const uint32_t f = lane < g ? see_flag(gflags + g - 1 - lane) : 0;
                const uint64_t whole = __ballot(f == 2), some = __ballot(f != 0);
                far = whole ? __builtin_ctzll(whole) : 64;
                const uint64_t between = far < 64 ? (1ull << far) - 1 : ~0ull;
                if ((far < 64 && (some & between) == between) || ++polls > kLooks) break;
            }
            // (a word may say less than its flag, for a moment, or more: any P on the way is as good)
            all = far < 64;
            bool known = false;
#pragma unroll 1
            for (int i0 = min(far, 63) & ~3; i0 >= 0; i0 -= 4) {
                uint64_t p[4];
                uint32_t at = ch * 8;
                asm volatile("" : "+v"(at));
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = look(sh.groups + max(g - 1 - i0 - i, 0) * D, at);
#pragma unroll
                for (int i = 3; i >= 0; --i)
                    if (i0 + i <= far) {
                        const uint32_t tag = tag_of(p[i]);
                        c = tag == kWhole ? pair_h(p[i]) : __fmaf_rn(pair_a(p[i]), c, pair_h(p[i]));
                        known = tag == kWhole || (known && tag != 0);
                    }
            }
            all = __all(known) && all;
            ++polls;
        }
        if (!all) c = __builtin_nanf("");
        if (pos == kGroup - 1) {
            if (Ag != 0.0f) leave(behind, kWhole, __fmaf_rn(Ag, c, Hg));
            raise_flag(gflags + g, 2);
        }
    }
    for (int i = 0; i < pos; ++i) c = through(pair_a(s_w[i * step]), pair_h(s_w[i * step]), c);
    return c;
}

// Words and flags to 0, the decay rates: 2.5 us for a small batch, most of it the launch, 5 to 6 for the 5 MB of
// 16384 x 2048 or 65536 x 1024.
__global__ __launch_bounds__(256) void recurrence_clear_kernel(RecShared s, int64_t n16, int D,
                                                               const float* __restrict__ lam, float rate) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t j = i; j < n16; j += (int64_t)gridDim.x * 256)
        reinterpret_cast<uint4*>(s.ticket)[j] = make_uint4(0, 0, 0, 0);
    for (int64_t j = i; j < D; j += (int64_t)gridDim.x * 256) s.k2[j] = decay_rate(lam[j], rate);
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

// A tile of 64 V channels: the at-th of the scan.
template <int V>
struct Place {
    int64_t t0;    // first token
    int order;     // its number in the scan
    int c0, ch;    // the first channel; the lane's first
    int real;      // tokens the tile really has
    bool act;      // false: a lane past the last channel, which computes the last ones again
    __device__ __forceinline__ Place(int at, int tile, int block, int64_t T, int D, int lane, bool reverse) {
        order = at;
        c0 = block * 64 * V;
        t0 = (reverse ? (T - 1) / tile - order : order) * tile;
        ch = min(c0 + lane * V, D - V);
        act = c0 + lane * V < D;
        real = (int)min((int64_t)tile, T - t0);
    }
};

// The bounds, in LDS where they fit.
constexpr int kCuLds = 2048;

template <int NT>
__device__ __forceinline__ void stage_bounds(const int32_t* __restrict__ cu, int S, int32_t* lds) {
    if (S >= kCuLds) return;
    for (int i = threadIdx.x; i <= S; i += NT) lds[i] = cu[i];
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
    RecShared sh;
};

// The kernel's argument, read again where it is asked for: what a loop over tiles keeps of it (and of
// addresses formed from it) from one tile to the next would take the registers of the tile.
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(4))) T& argument() {
    auto p = (const __attribute__((address_space(4))) T*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

// The workgroup's block of channels, as many workgroups for each.  Tiles of a block end in the order of the
// scan, so its workgroups move in step; each XCD and each CU holds workgroups of different blocks, whose steps
// differ, so that some compute while others load (65536 x 1024 took 215 us with a block on one XCD when it
// took 165 so).
__device__ __forceinline__ int my_block(int blocks) {
    // Workgroups go to the 8 XCDs in turn, and there to 32 CUs: `at` numbers them XCD by XCD, and a shift
    // after every 32 or more (whole turns of the blocks) keeps a CU's next one off the same block.
    const int n = gridDim.x, xcd = blockIdx.x % 8, at = xcd * (n / 8) + min(xcd, n % 8) + blockIdx.x / 8;
    return (at + at / ((31 / blocks + 1) * blocks)) % blocks;
}

// The lane's decay rates.
template <int V, typename Args>
__device__ __forceinline__ void decay_rates(const Args& arg, int block, float (&k2)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int ch = min(block * 64 * V + (int)(threadIdx.x & 63) * V, arg.D - V) + k;
        k2[k] = arg.sh.k2 ? arg.sh.k2[ch] : decay_rate(arg.lam[ch], arg.rate);
    }
}

// Whether they all stay below kSmall (decays above 0.88 even at open gates): those take fewer instructions, which
// the waits hide.  16384 x 2048 bf16 with rates below it 73 us and 116 back, past it 74 and 120.
template <int V>
__device__ __forceinline__ bool all_small(const float (&k2)[V]) {
    bool small = true;
#pragma unroll
    for (int k = 0; k < V; ++k) small = small && k2[k] < kSmall;
    return __all(small);
}

// The look back over the workgroup's 64 V slots (a lane's V channels side by side), a slot a lane of
// V waves: the waves' pairs (s_a, s_h) in the scan's order make the tile's, and s_c gets the state
// before it.
template <int V, int WAVES, typename Shared>
__device__ __forceinline__ void look_back(const Shared& sh, int order, int tiles, int c0, int D, bool reverse, int slot,
                                          const float (&s_a)[WAVES][64 * V], const float (&s_h)[WAVES][64 * V],
                                          float (&s_c)[64 * V], uint64_t* s_w) {
    const int ch = min(c0 + slot / V * V, D - V) + slot % V;
    float A = 1.0f, H = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const int w = reverse ? WAVES - 1 - i : i;
        const float aw = s_a[w][slot];
        H = through(aw, s_h[w][slot], H);
        A = joined(A, aw);
    }
    const int part = __builtin_amdgcn_readfirstlane((c0 + slot) / 64);
    s_c[slot] = sh.ticket ? state_before(sh, order, tiles, D, part, ch, A, H, s_w + slot, 64 * V)
                          : 0.0f;
}

// (A, H) of the lane's channels over the waves from `first`, `n` of them, in steps of `step`.
template <int V, int WAVES>
__device__ __forceinline__ void through_waves(const float (&s_a)[WAVES][64 * V], const float (&s_h)[WAVES][64 * V],
                                              int lane, int first, int n, int step, float (&A)[V], float (&H)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
    for (int i = 0; i < n; ++i) {
        const int w = first + i * step;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float a = s_a[w][lane * V + k];
            H[k] = through(a, s_h[w][lane * V + k], H[k]);
            A[k] = joined(A[k], a);
        }
    }
}

// Workgroups take tiles of kTile tokens and 64 V channels, V a lane, in the order of the scan; each wave
// takes R of the tile's tokens.  Bound by waiting for the tiles before: 65536 x 1024 bf16 (537 MB) 134 us, 112
// in a copy that does not wait, 106 at a copy's rate; 40796 x 2048 150, 127 and 132; 16384 x 2048 73, 63 and 53, f32
// 118, 111 and 106.  As fast: 16 tokens a wave and two workgroups a CU, 8 tokens and three.  Slower: the next
// tile's inputs on their way and its pair left before this tile's state is looked up (that takes 256 registers, two
// waves a SIMD: 220 us where this took 150); a ticket taken before the wait (168 for 136), as it then lies with a
// workgroup that waits and holds all later tiles up.  The bf16 form spills 3 of its 128 registers.
template <int DT, int V, int R>
__global__ __launch_bounds__(64 * (kTile / R), 4) void recurrence_kernel(RecFwd arg) {
    constexpr int WAVES = kTile / R, NT = 64 * WAVES;
    __shared__ int32_t s_cu[kCuLds];
    __shared__ uint64_t s_w[(kGroup - 1) * 64 * V];
    __shared__ int32_t s_seq[kTile];
    __shared__ int s_next;
    __shared__ float s_c[64 * V], s_a[2][WAVES][64 * V], s_h[2][WAVES][64 * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = (int)((arg.T - 1) / kTile + 1), block = my_block((arg.D - 1) / (64 * V) + 1);
    // (ticket, rates and bounds on their way at once)
    int first = 0;
    if (threadIdx.x == 0 && arg.sh.ticket) first = (int)atomicAdd(arg.sh.ticket + block * 16, 1u);
    float k2[V];
    decay_rates<V>(arg, block, k2);
    stage_bounds<NT>(arg.cu, arg.S, s_cu);
    if (threadIdx.x == 0) s_next = first;
    __syncthreads();
    int at = __builtin_amdgcn_readfirstlane(s_next);
    const bool small = all_small<V>(k2);
    const bool again = (int64_t)gridDim.x < (int64_t)tiles * ((arg.D - 1) / (64 * V) + 1);  // (else a tile each)
    for (int turn = 0; at < tiles; turn ^= 1) {
        const auto& P = argument<RecFwd>();
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const Place<V> p(at, kTile, block, P.T, P.D, lane, false);
        const int ch = p.ch;
        const uint32_t off = ch * (DT == NSOSX_F32 ? 4 : 2);
        Pair<DT, V> x[R], r[R], g[R];
        {
            const Rows vx = tile_rows<DT>(P.x, P.xs, p.t0), vr = tile_rows<DT>(P.rg, P.rs, p.t0),
                       vg = tile_rows<DT>(P.ig, P.is, p.t0);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int t = min(wave * R + j, p.real - 1);
                r[j].load(vr, off, t);
                g[j].load(vg, off, t);
                x[j].load(vx, off, t);
            }
        }
        Tokens tok;  // (a search of its own for either memory: one through a flat address would wait for the inputs)
        if (P.S < kCuLds) tok = find_tokens<R>(s_cu, P.S, lane, p.t0 + wave * R, P.T, s_seq + wave * R);
        else tok = find_tokens<R>(P.cu, P.S, lane, p.t0 + wave * R, P.T, s_seq + wave * R);
        const bool plain = tok.template plain<R>();
        float a[R][V], u[R][V];
        auto gates = [&](auto fits) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                r[j].forget();
                g[j].forget();
                x[j].forget();
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float q = k2[k] * sigmoid_of(exp_neg(r[j].get(k)));
                    a[j][k] = __builtin_amdgcn_exp2f(-q);
                    u[j][k] = __builtin_amdgcn_sqrtf(one_less_square<decltype(fits)::value>(q, a[j][k])) *
                              (sigmoid_of(exp_neg(g[j].get(k))) * x[j].get(k));
                }
                __builtin_amdgcn_sched_barrier(0);  // token after token, or all of them are half done at once
            }
        };
        if (small) gates(std::true_type{});
        else gates(std::false_type{});
        float A[V], H[V];
#pragma unroll
        for (int k = 0; k < V; ++k) A[k] = 1.0f, H[k] = 0.0f;
        auto local = [&](auto borders) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const bool start = decltype(borders)::value && (tok.starts >> j & 1);
                if (start) take_state<V>(P.initial, s_seq[wave * R + j], P.D, ch, H);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
                    A[k] = start ? 0.0f : A[k] * a[j][k];
                }
            }
        };
        if (plain) local(std::false_type{});
        else local(std::true_type{});
        if (!tok.starts) {
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = fmaxf(A[k], kLeast);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) s_a[turn][wave][lane * V + k] = A[k], s_h[turn][wave][lane * V + k] = H[k];
        __syncthreads();
        if (wave < V) look_back<V, WAVES>(P.sh, p.order, tiles, p.c0, P.D, false, wave * 64 + lane, s_a[turn], s_h[turn], s_c, s_w);
        // (the waves before this one in the tile, meanwhile)
        through_waves<V>(s_a[turn], s_h[turn], lane, 0, wave, 1, A, H);
        __syncthreads();
        float h[V];
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = through(A[k], H[k], s_c[lane * V + k]);
        if (wave * R % kKept == 0 && P.carry && wave * R < p.real && p.act)
            put_state<V>(P.carry, (int)((p.t0 + wave * R) / kKept), P.D, ch, h);
        const Rows vy = tile_rows<DT>(P.y, P.ys, p.t0);
        auto apply = [&](auto borders) {
            constexpr bool B = decltype(borders)::value;
            const float zero[V] = {};
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int t = wave * R + j;
                if (B && !(tok.inside >> j & 1)) {
                    if (P.rest && t < p.real && p.act) Pair<DT, V>::store(vy, off, t, zero);
                    continue;
                }
                if (B && (tok.starts >> j & 1)) take_state<V>(P.initial, s_seq[wave * R + j], P.D, ch, h);
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] = __fmaf_rn(a[j][k], h[k], u[j][k]);
                if (p.act) Pair<DT, V>::store(vy, off, t, h);
                if (B && (tok.ends >> j & 1) && P.final) {
                    const int seq = s_seq[wave * R + j];
                    if (p.act) put_state<V>(P.final, seq, P.D, ch, h);
                }
            }
        };
        if (plain) apply(std::false_type{});
        else apply(std::true_type{});
        if (threadIdx.x == 0) s_next = again ? (int)atomicAdd(P.sh.ticket + block * 16, 1u) : tiles;
        __syncthreads();
        at = __builtin_amdgcn_readfirstlane(s_next);
        if (p.order == 0 && P.final) empty_states<V, NT>(P.cu, P.S, P.D, ch, p.act, P.initial, P.final);
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
    RecShared sh;
};

// The same from the last tile to the first.  With q = g / log 2, w = a q and b2 = 1 - a^2:
//   e = dh (s x a w / beta - w h_before), in units of log 2
// (where beta goes to 0 so does w, faster).  Tiles of 64 tokens, 8 a wave: four values an element have to
// stay in registers over the wait.  16384 x 2048 bf16 (470 MB) 116 us, 98 in a copy that does not wait, 93
// at a copy's rate (77 vector instructions a place, 9 of them exponentials, roots and reciprocals); f32 172 and
// 161, at a copy's rate 185 (part of it stays in the 256 MB cache).  2 or 3 registers are spilled; with 1 - a^2 kept
// too 31, and 159 us where this took 134.
template <int DT, int V, int R>
__global__ __launch_bounds__(64 * (kKept / R), V == 1 ? 6 : 4) void recurrence_bwd_kernel(RecBwd arg) {
    constexpr int WAVES = kKept / R, NT = 64 * WAVES;
    __shared__ int32_t s_cu[kCuLds];
    __shared__ uint64_t s_w[(kGroup - 1) * 64 * V];
    __shared__ int32_t s_seq[kKept];
    __shared__ int s_next;
    __shared__ float s_c[64 * V], s_a[WAVES][64 * V], s_h[WAVES][64 * V], s_b[WAVES][64 * V],
        s_m[WAVES][64 * V], s_e[WAVES][64 * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = (int)((arg.T - 1) / kKept + 1), block = my_block((arg.D - 1) / (64 * V) + 1);
    // (ticket, rates and bounds on their way at once)
    int first = 0;
    if (threadIdx.x == 0 && arg.sh.ticket) first = (int)atomicAdd(arg.sh.ticket + block * 16, 1u);
    float k2[V];
    decay_rates<V>(arg, block, k2);
    stage_bounds<NT>(arg.cu, arg.S, s_cu);
    if (threadIdx.x == 0) s_next = first;
    __syncthreads();
    int at = __builtin_amdgcn_readfirstlane(s_next);
    const bool small = all_small<V>(k2);
    const bool again = (int64_t)gridDim.x < (int64_t)tiles * ((arg.D - 1) / (64 * V) + 1);  // (else a tile each)
    while (at < tiles) {
        const auto& P = argument<RecBwd>();
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const Place<V> p(at, kKept, block, P.T, P.D, lane, true);
        const int ch = p.ch;
        const uint32_t off = ch * (DT == NSOSX_F32 ? 4 : 2);
        // kept over the wait: a, u (then the state before each token), e^-rg, e^-ig, x and dy as loaded
        float a[R][V], u[R][V], er[R][V], eg[R][V], h[V];
        Pair<DT, V> x[R], d[R];
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
            take_state<V>(P.carry, (int)(p.t0 / kKept), P.D, ch, h);
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    er[j][k] = exp_neg(r[j].get(k));
                    eg[j][k] = exp_neg(g[j].get(k));
                }
        }
        Tokens tok;  // (a search of its own for either memory: one through a flat address would wait for the inputs)
        if (P.S < kCuLds) tok = find_tokens<R>(s_cu, P.S, lane, p.t0 + wave * R, P.T, s_seq + wave * R);
        else tok = find_tokens<R>(P.cu, P.S, lane, p.t0 + wave * R, P.T, s_seq + wave * R);
        const bool plain = tok.template plain<R>();
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
        float A[V], H[V], B[V], M[V];
#pragma unroll
        for (int k = 0; k < V; ++k) A[k] = B[k] = 1.0f, H[k] = M[k] = 0.0f;
        auto local = [&](auto borders) {
            constexpr bool BORDERS = decltype(borders)::value;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const bool start = BORDERS && (tok.starts >> j & 1);
                if (start) take_state<V>(P.initial, s_seq[wave * R + j], P.D, ch, H);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    H[k] = __fmaf_rn(a[j][k], H[k], u[j][k]);
                    A[k] = start ? 0.0f : A[k] * a[j][k];
                }
            }
#pragma unroll
            for (int j = R - 1; j >= 0; --j) {
                const bool end = BORDERS && (tok.ends >> j & 1), out = BORDERS && !(tok.inside >> j & 1);
                if (end) take_state<V>(P.dfinal, s_seq[wave * R + j], P.D, ch, M);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    M[k] = out ? 0.0f : a[j][k] * (d[j].get(k) + M[k]);
                    if (BORDERS) B[k] = end || out ? 0.0f : B[k] * a[j][k];
                }
            }
        };
        if (plain) local(std::false_type{});
        else local(std::true_type{});
        if (!tok.starts) {
#pragma unroll
            for (int k = 0; k < V; ++k) A[k] = fmaxf(A[k], kLeast);
        }
        if (plain) {
#pragma unroll
            for (int k = 0; k < V; ++k) B[k] = A[k];
        } else if (!tok.ends && tok.inside == (1u << R) - 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) B[k] = fmaxf(B[k], kLeast);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            s_a[wave][lane * V + k] = A[k], s_h[wave][lane * V + k] = H[k];
            s_b[wave][lane * V + k] = B[k], s_m[wave][lane * V + k] = M[k];
        }
        __syncthreads();
        if (wave >= WAVES - V)
            look_back<V, WAVES>(P.sh, p.order, tiles, p.c0, P.D, true, (wave - (WAVES - V)) * 64 + lane, s_b, s_m, s_c, s_w);
        through_waves<V>(s_a, s_h, lane, 0, wave, 1, A, H);
        through_waves<V>(s_b, s_m, lane, WAVES - 1, WAVES - 1 - wave, -1, B, M);
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = through(A[k], H[k], h[k]);
        // u becomes the state before each token
        auto states = [&](auto borders) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (decltype(borders)::value && (tok.starts >> j & 1))
                    take_state<V>(P.initial, s_seq[wave * R + j], P.D, ch, h);
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
        float m[V], e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            m[k] = through(B[k], M[k], s_c[lane * V + k]);
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
                if (BORDERS && !(tok.inside >> j & 1)) {
                    if (P.rest && t < p.real && p.act) {
                        Pair<DT, V>::store(vx, off, t, zero);
                        Pair<DT, V>::store(vr, off, t, zero);
                        Pair<DT, V>::store(vg, off, t, zero);
                    }
                    continue;
                }
                if (BORDERS && (tok.ends >> j & 1)) take_state<V>(P.dfinal, s_seq[wave * R + j], P.D, ch, m);
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
                if (BORDERS && (tok.starts >> j & 1) && P.dinitial) {
                    const int seq = s_seq[wave * R + j];
                    if (p.act) put_state<V>(P.dinitial, seq, P.D, ch, m);
                }
            }
        };
        if (!plain) apply(std::true_type{}, std::false_type{});
        else if (small) apply(std::false_type{}, std::true_type{});
        else apply(std::false_type{}, std::false_type{});
#pragma unroll
        for (int k = 0; k < V; ++k) s_e[wave][lane * V + k] = e[k];
        if (threadIdx.x == 0) s_next = again ? (int)atomicAdd(P.sh.ticket + block * 16, 1u) : tiles;
        __syncthreads();
        at = __builtin_amdgcn_readfirstlane(s_next);
        if (wave == 0 && p.act) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                for (int w = 1; w < WAVES; ++w) e[k] += s_e[w][lane * V + k];  // (next written two barriers on)
            put_state<V>(P.dlam_part, (int)(p.t0 / kKept), P.D, ch, e);
        }
        if (p.order == 0 && P.dinitial) empty_states<V, NT>(P.cu, P.S, P.D, ch, p.act, P.dfinal, P.dinitial);
    }
}

// dlam = sigmoid(lam) / softplus(lam) * sum_t e, e in units of log 2: the tiles' sums in a fixed order (16
// channels a workgroup, 64 runs of tiles: a short chain of loads, as the sums are few).  256 tiles x 2048
// channels 4 us, with 64 channels a workgroup 8.
__global__ __launch_bounds__(1024) void recurrence_dlam_kernel(const float* __restrict__ part, int tiles,
                                                               int D, const float* __restrict__ lam,
                                                               float* __restrict__ dlam) {
    __shared__ float s[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 16 + (lane & 15);
    const float* p = part + min(c, (int64_t)D - 1);
    float sum = 0.0f;
#pragma unroll 8
    for (int i = threadIdx.x >> 4; i < tiles; i += 64) sum += p[(int64_t)i * D];
    sum += lane_xor<16>(sum);
    sum += lane_xor<32>(sum);
    if (lane < 16) s[wave][lane] = sum;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= D) return;
    for (int w = 1; w < 16; ++w) sum += s[w][lane];
    // sigmoid / softplus goes to 1 as both go to e^lam
    const float l = lam[c], en = expf(-fabsf(l));
    const float sig = l < 0.0f ? en / (1.0f + en) : 1.0f / (1.0f + en);
    const float sp = fmaxf(l, 0.0f) + log1pf(en);
    dlam[c] = sum * kLn2 * (sp == 0.0f ? 1.0f : sig / sp);
}

// One token per row: a thread per channel and run of kStepRows rows, which share the channel's decay rate (a
// logarithm and two exponentials).  Bound by the launch (8 x 2048) or by memory: 1000 x 2559 f32, 61 MB, in
// a call of 11.5 us, 12 at a copy's rate (part of it stays in the 256 MB cache).
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

// Whether a block of n bytes (states, rates) and a view's rows share an element.
static bool block_meets(const void* b, int64_t n, const void* v, int64_t vs, int64_t rows, int64_t D, int64_t size) {
    if (!b || !v || rows <= 0 || n <= 0 || !overlaps(b, n, v, ((rows - 1) * vs + D) * size)) return false;
    if (rows == 1) return true;
    const int64_t row = vs * size;
    int64_t off = (static_cast<const char*>(b) - static_cast<const char*>(v)) % row;
    if (off < 0) off += row;
    return off < D * size || off + n > row;
}

static const char* rec_check(int S, int64_t T, int D, int dtype, float rate) {
    if (S < 0 || T < 0 || D <= 0) return "need sequences >= 0, tokens >= 0 and dim > 0";
    if (!valid_dtype(dtype)) return "bad dtype";
    if (!(rate > 0.0f) || rate > 3.0e38f) return "rate must be finite and > 0";
    return nullptr;
}

static std::atomic<int> g_looks{kLooks};

// What the tiles share, in the workspace: ticket (16 bytes), words, flags, decay rates; nothing for one
// tile in time.
static RecShared rec_shared(int64_t tiles, int D, void* workspace, int64_t* clear, int64_t* bytes) {
    RecShared s{};
    const int64_t groups = (tiles - 1) / kGroup + 1, parts = ((int64_t)D + 63) / 64 + 1;
    *clear = *bytes = 0;
    if (tiles <= 1) return s;
    char* at = static_cast<char*>(workspace);
    int64_t n = 64 * parts;
    s.ticket = reinterpret_cast<uint32_t*>(at);
    s.words = reinterpret_cast<uint64_t*>(at + n);
    n += tiles * D * 8;
    s.groups = reinterpret_cast<uint64_t*>(at + n);
    n += groups * D * 8;
    s.flags = reinterpret_cast<uint32_t*>(at + n);
    n += parts * tiles * 4;
    s.gflags = reinterpret_cast<uint32_t*>(at + n);
    n = (n + parts * groups * 4 + 15) / 16 * 16;
    *clear = n / 16;
    s.k2 = reinterpret_cast<float*>(at + n);
    s.spent = kLooks - g_looks.load(std::memory_order_relaxed);
    *bytes = n + ((int64_t)D * 4 + 15) / 16 * 16;
    return s;
}

static int64_t rec_shared_bytes(int64_t tiles, int D) {
    int64_t clear, bytes;
    rec_shared(tiles, D, nullptr, &clear, &bytes);
    return bytes;
}

static RecShared start_shared(int64_t tiles, int D, const float* lam, float rate, void* workspace, hipStream_t st) {
    int64_t clear, bytes;
    const RecShared s = rec_shared(tiles, D, workspace, &clear, &bytes);
    if (!bytes) return s;
    const int64_t blocks = (clear + 1023) / 1024;
    hipLaunchKernelGGL(recurrence_clear_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st,
                       s, clear, D, lam, rate);
    return s;
}

// Workgroups: as many as the card holds at once, the same number for every block of channels.
static unsigned rec_grid(int64_t tiles, int D, int V, int resident) {
    const int64_t blocks = (D - 1) / (64 * V) + 1, each = resident / blocks;
    return (unsigned)(blocks * (each < 1 ? 1 : each < tiles ? each : tiles));
}

// bf16: two channels a lane, f32 one (64 channels are a full line there, and the registers carry more
// workgroups).  16384 x 2048 f32 with one 118 us and 172 back, with two 1.45 times as long when both were there; bf16
// with two 73 and 116, with one 79 and 120 (65536 x 1024: 134 and 153).
template <int DT, int V>
static void launch_recurrence(const RecFwd& p, hipStream_t st) {
    hipLaunchKernelGGL((recurrence_kernel<DT, V, 16>), dim3(rec_grid(rec_tiles(p.T, kTile), p.D, V, 512)),
                       dim3(64 * (kTile / 16)), 0, st, p);
}

template <int DT, int V>
static void launch_recurrence_bwd(const RecBwd& p, hipStream_t st) {
    hipLaunchKernelGGL((recurrence_bwd_kernel<DT, V, 8>),
                       dim3(rec_grid(rec_tiles(p.T, kKept), p.D, V, V == 1 ? 768 : 512)), dim3(64 * (kKept / 8)),
                       0, st, p);
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

extern "C" int nsosx_gated_recurrence_looks(int looks) {
    if (looks < 0) return g_looks.load(std::memory_order_relaxed);
    return g_looks.exchange(looks < kLooks ? looks : kLooks, std::memory_order_relaxed);
}

extern "C" int64_t nsosx_gated_recurrence_workspace(int T, int D) {
    if (T <= 0 || D <= 0) return 0;
    const int64_t bytes = rec_shared_bytes(rec_tiles(T, kTile), D);
    return bytes < 16 ? 16 : bytes;
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
    if (!x || !rg || !ig || !y || !workspace)
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
    if (block_meets(initial_state, sd * 4, y, y_stride, T, D, size) || block_meets(lam, (int64_t)D * 4, y, y_stride, T, D, size))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence: y overlaps an input");
    RecFwd p{x, rg, ig, x_stride, rg_stride, ig_stride, lam, rate, cu_seqlens, S, T, D, zero_rest,
             initial_state, y, y_stride, final_state, carry,
             start_shared(rec_tiles(T, kTile), D, lam, rate, workspace, st)};
    if (act_dtype == NSOSX_F32) {
        launch_recurrence<NSOSX_F32, 1>(p, st);
    } else {
        if (D > 1) launch_recurrence<NSOSX_BF16, 2>(p, st);
        else launch_recurrence<NSOSX_BF16, 1>(p, st);
    }
    return check_launch("gated_recurrence");
}

extern "C" int64_t nsosx_gated_recurrence_backward_workspace(int T, int D) {
    if (T <= 0 || D <= 0) return 0;
    return rec_shared_bytes(rec_tiles(T, kKept), D) + rec_tiles(T, kKept) * D * 4;
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
        if (block_meets(initial_state, sd * 4, out[o], out_s[o], T, D, size) ||
            block_meets(dfinal, sd * 4, out[o], out_s[o], T, D, size) ||
            block_meets(carry, rec_tiles(T, kKept) * D * 4, out[o], out_s[o], T, D, size) ||
            block_meets(lam, (int64_t)D * 4, out[o], out_s[o], T, D, size))
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
             dinitial, reinterpret_cast<float*>(static_cast<char*>(workspace) + rec_shared_bytes(rec_tiles(T, kKept), D)),
             start_shared(rec_tiles(T, kKept), D, lam, rate, workspace, st)};
    if (act_dtype == NSOSX_F32) {
        launch_recurrence_bwd<NSOSX_F32, 1>(p, st);
    } else {
        if (D > 1) launch_recurrence_bwd<NSOSX_BF16, 2>(p, st);
        else launch_recurrence_bwd<NSOSX_BF16, 1>(p, st);
    }
    hipLaunchKernelGGL(recurrence_dlam_kernel, dim3((D + 15) / 16), dim3(1024), 0, st, p.dlam_part,
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
    // (element for element the states may lie over f32 views: a thread reads its own before it writes it)
    const void* seen[4] = {x, rg, ig, y};
    const int64_t seen_s[4] = {x_stride, rg_stride, ig_stride, y_stride};
    for (int i = 0; i < 4; ++i) {
        const bool dense = size == 4 && (rows == 1 || seen_s[i] == D);
        if (!(dense && seen[i] == state_out) && block_meets(state_out, n, seen[i], seen_s[i], rows, D, size))
            return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: state_out overlaps an input or y");
    }
    if (!(size == 4 && (rows == 1 || y_stride == D) && y == state) && block_meets(state, n, y, y_stride, rows, D, size))
        return fail(NSOSX_ERR_INVALID, "gated_recurrence_step: y overlaps state");
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
