// Scored expert routing on gfx950: softmax or sigmoid scores, a balance bias that takes part in
// the choice only, expert groups, top-k, renormalised and scaled weights, the dispatch to
// expert segments, and the gradient of the logits from that of the weights.
#include "common.hpp"

namespace nsosx {

constexpr int kScoredMaxExperts = 512, kScoredMaxK = 16, kScoredMaxGroups = 16;
constexpr int kScoredMaxRows = (1 << 28) - 64;  // 16 threads each: a launch holds fewer than 2^32

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
    int32_t* block_counts;   // workspace [E, blocks]; where by_block, bytes [blocks, words of 4]
    int by_block;
    int size, lanes, run;    // experts of a group, lanes that share them (a power of two), of a lane
    int pitch;               // of a row in LDS, floats
};

// ---- sixteen lanes per row -----------------------------------------------------
// A row's experts lie on the 16 lanes of a DPP row, so that four rows share a wave and every
// reduction over a row is four rotations: expert 16 v + l in value v of lane l or, where the
// choice is limited to groups, each group on `lanes` neighbouring lanes of its own, a run of its
// experts each, so that a group's score is a reduction over those lanes.  The row then goes through
// LDS: loaded in runs, 64 lanes meet 64 cache lines a time (16384 rows of 256: 7 us more).

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
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

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

// This lane's values of a row of E floats, expert 16 v + l in value v, -inf past E or where the row
// is not live.  (Every load is made, from the last expert where there is none: a branch around
// each would wait for each.)
template <int V, int DT>
__device__ __forceinline__ void row_values(const void* x, int64_t base, int E, bool live, float (&c)[V]) {
    const int l = threadIdx.x & 15;
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = load_act<DT>(x, base + min(16 * v + l, E - 1));
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = live && 16 * v + l < E ? c[v] : -INFINITY;
}

// Floats first .. first + n - 1 of a row in LDS, behind them -inf (or, where FILL is not, any value of
// the run); in 16-byte pieces where every lane's run allows it.
template <int V, bool FILL = true>
__device__ __forceinline__ void run_values(const float* row, int first, int n, bool pieces, float (&c)[V]) {
    if (pieces && V >= 4) {
#pragma unroll
        for (int v = 0; v + 3 < V; v += 4) {
            const float4 f = *reinterpret_cast<const float4*>(row + first + (v < n ? v : 0));
            c[v] = f.x; c[v + 1] = f.y; c[v + 2] = f.z; c[v + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = row[first + (v < n ? v : 0)];
    }
    if constexpr (FILL) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = v < n ? c[v] : -INFINITY;
    }
}

template <int CTRL>
__device__ __forceinline__ void join2(float& a, float& b) {
    const float oa = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(a), CTRL, 0xF, 0xF, true));
    const float ob = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(b), CTRL, 0xF, 0xF, true));
    b = fmaxf(fminf(a, oa), fmaxf(b, ob));
    a = fmaxf(a, oa);
}
template <int N>
__device__ __forceinline__ void outranked(float s, int q, int& lanes) {
    const float o = ror16<N>(s);
    const int oq = ror16<N>(q);
    lanes += o > s || (o == s && oq < q) ? 1 : 0;
}
__device__ __forceinline__ float row_min(float v) { return -row_max(-v); }

// Whether this lane's group is one of the `keep` best (ties to the lower group), from the values of
// its experts; -inf, an unavailable expert, adds nothing.  err: the scores' error.  clear: whether
// every group that stays is above every one that goes by more than both groups' errors.  Those are each
// group's own: its two scores', and, in units u = 2^-23, half a unit of each value (the sum with the
// bias), of the group's sum, and of that less or plus `room`, together below 1.5 u (|a| + |b|).  Where a
// group's second value holds a mask that is large and finite (-1e4, say), that is far more than
// the row's largest value would give.
template <int V>
__device__ __forceinline__ bool group_stays(const RouteScored& p, const float (&c)[V], int q, float err,
                                            bool& clear) {
    const float none = -INFINITY;
    float a = none, b = none;  // the group's two largest
#pragma unroll
    for (int v = 0; v < V; ++v) {
        b = fmaxf(b, fminf(a, c[v]));
        a = fmaxf(a, c[v]);
    }
    if (p.lanes >= 2) join2<0xB1>(a, b);   // lane l ^ 1
    if (p.lanes >= 4) join2<0x4E>(a, b);   // lane l ^ 2
    if (p.lanes >= 8) join2<0x141>(a, b);  // lane l ^ 7: the other four of eight
    const bool two = p.best == 2 && b > none;
    float s = two ? a + b : a;
    if (q >= p.groups) s = none;
    int better = 0;  // lanes of better groups
    outranked<1>(s, q, better); outranked<2>(s, q, better); outranked<3>(s, q, better);
    outranked<4>(s, q, better); outranked<5>(s, q, better); outranked<6>(s, q, better);
    outranked<7>(s, q, better); outranked<8>(s, q, better); outranked<9>(s, q, better);
    outranked<10>(s, q, better); outranked<11>(s, q, better); outranked<12>(s, q, better);
    outranked<13>(s, q, better); outranked<14>(s, q, better); outranked<15>(s, q, better);
    const bool in = q < p.groups && better < p.keep * p.lanes;
    // (each term by itself: |a| + |b| may pass the largest float)
    const float room = 2.0f * err + 0x1p-22f * fabsf(a) + (two ? 0x1p-22f * fabsf(b) : 0.0f);
    const float low = row_min(in ? s - room : INFINITY);
    // (a group without an available expert, which ranks last, has s and room infinite)
    clear = low > row_max(in || s == none ? none : s + room);
    return in;
}

// exp(x) to a unit in 64 bits: x = n ln 2 + r with |r| <= ln 2 / 2, the Taylor sum of exp(r) to
// r^13 (the next term is below 2^-57), times 2^n.
__device__ __forceinline__ double exp_of(double x) {
    x = fmin(fmax(x, -800.0), 800.0);  // 0 and infinity past either end
    const double n = rint(x * 0x1.71547652b82fep+0);
    double r = fma(-n, 0x1.62e42fefa39efp-1, x);
    r = fma(-n, 0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

// Whether lane l - N of the row has a larger value (or the same one and a lower index).
template <int N>
__device__ __forceinline__ void outranked64(double v, int e, int& rank) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = ror16<N>((uint32_t)u), hi = ror16<N>((uint32_t)(u >> 32));
    const double o = __builtin_bit_cast(double, lo | (hi << 32));
    const int oe = ror16<N>(e);
    rank += o > v || (o == v && oe < e) ? 1 : 0;
}
// Of rank << 16 | index in each lane, the one whose rank is this lane's number.
template <int N>
__device__ __forceinline__ void ranked_here(uint32_t at, int l, uint32_t& got) {
    const uint32_t o = ror16<N>(at);
    got = (int)(o >> 16) == l ? o : got;
}

// The maximum and the scores' sum of a softmax row (unavailable experts are -inf).
template <int V>
__device__ __forceinline__ void softmax_stats(const float (&x)[V], float& mx, float& sum) {
    mx = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) mx = fmaxf(mx, x[v]);
    mx = row_max(mx);
    sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += x[v] == -INFINITY ? 0.0f : expf(x[v] - mx);  // a NaN stays
    sum = row_sum(sum);
}

// Batcher's odd-even merge sort, descending, of N keys from LO.
template <int A, int B, int V>
__device__ __forceinline__ void order_pair(uint32_t (&key)[V]) {
    const uint32_t a = key[A], b = key[B];
    key[A] = a > b ? a : b;
    key[B] = a > b ? b : a;
}
template <int I, int END, int R, int V>
__device__ __forceinline__ void order_pairs(uint32_t (&key)[V]) {
    if constexpr (I + R < END) {
        order_pair<I, I + R>(key);
        order_pairs<I + 2 * R, END, R>(key);
    }
}
template <int LO, int N, int R, int V>
__device__ __forceinline__ void merge_keys(uint32_t (&key)[V]) {
    if constexpr (2 * R < N) {
        merge_keys<LO, N, 2 * R>(key);
        merge_keys<LO + R, N, 2 * R>(key);
        order_pairs<LO + R, LO + N, R>(key);
    } else {
        order_pair<LO, LO + R>(key);
    }
}
template <int LO, int N, int V>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[V]) {
    if constexpr (N > 1) {
        sort_keys<LO, N / 2>(key);
        sort_keys<LO + N / 2, N / 2>(key);
        merge_keys<LO, N, 1>(key);
    }
}

// The choice by 32-bit scores, with a proof that it is the one of 64 bits: every value becomes a
// 32-bit key, its distance from a point below the row's largest in fixed point (2 for scores with a
// bias, 32 for logits, whose order is that of scores without one) above the complement of its
// index, each lane sorts its keys, and k + 1 rounds take the largest of the row's 16 first ones.
// The choice stands where the fixed-point values of neighbours in that order differ by more than
// the scores' error.  Where they do not (about 7 of 10^4 rows of 256 sigmoid scores with a bias), but
// the k + 1 largest are apart from all others, those are put in order in 64 bits, one a lane.
// What is left (groups too close together, more values than that, values outside the window, a NaN in
// the row) the whole wave chooses in 64 bits, a row at a time (select_wave).  bfloat16 logits make
// exact keys.
//
// What it takes is instructions: 16384 rows of 256 experts in 8 groups, sigmoid scores and a bias,
// are 17 MB (3.3 us) and 14 .. 15 us, 12 without the rows that 32 bits cannot decide; vector
// instructions are issued in 77 % of the clocks.  (k rounds of a 64-bit maximum over every row took 41;
// select_wave alone for those rows, 4 us of one wave while the launch waits for it, 18.)  Where
// select_wave has every row, a call of 20 us takes 42 .. 48: all values equal, scores of 2e-9 that
// only their sums in a group part, a mask of -1e4 on all experts of each group but one.
//
// Errors, in units u = 2^-23: a sigmoid by exp2 and reciprocal of one unit each is off by s (1 - s)
// (|x| / 2 + 1) + 1.5 s, below 1.7 u.  A softmax score p = e / sum: e by |x - max| + 1 of itself,
// the sum by (V + 4) / 2 + 1 and the weighted mean of |x - max|, at most ln 512, reciprocal and
// product 1.5, and p |x - max| <= 0.37 of the largest p: below (13 + V / 2) u of that.  The sum with
// the bias by half a unit of the value.
//
// Expert index of choice l in lane l (-1: none), where `sure`.  G: limited to groups.
// s_row, s_bias (G): this row's place in LDS, the biases there.
template <int V, int DT, bool G>
__device__ __forceinline__ int select_fast(const RouteScored& p, int64_t row, bool live, float* s_row,
                                           const float* s_bias, bool& sure) {
    constexpr int IB = V == 2 ? 5 : V == 4 ? 6 : V == 8 ? 7 : V == 16 ? 8 : 9;  // bits of an index
    constexpr int NB = 32 - IB;
    constexpr uint32_t kIndex = (1u << IB) - 1;
    const float none = -INFINITY;
    const int l = threadIdx.x & 15;
    const int lanes = G ? max(p.lanes, 1) : 16;
    const int q = G ? min(l / lanes, p.groups - 1) : 0, at = G ? l % lanes * p.run : l;
    const bool real = !G || (p.lanes > 0 && l / lanes < p.groups);  // a lane with experts
    // this lane's experts: first + v step
    const int first = G ? q * p.size + (at < p.size ? at : 0) : l, step = G ? 1 : 16;
    const bool scored = p.bias || (G && p.best == 2);
    float x[V], c[V], b[V];
    bool odd = false;  // a NaN, or an infinite logit of a softmax
    row_values<V, DT>(p.logits, row * p.stride, p.E, live, x);
    if (G) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (16 * v + l < p.E) s_row[16 * v + l] = x[v];
        // the wave reads what its own lanes wrote
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int n = real ? min(p.run, p.size - at) : 0;
        const bool pieces = p.size % 4 == 0 && p.run % 4 == 0;
        run_values<V>(s_row, first, n, pieces, x);
        if (p.bias) run_values<V, false>(s_bias, first, n, pieces, b);
    } else if (p.bias) {
        row_values<V, NSOSX_F32>(p.bias, 0, p.E, true, b);
    }
    float err = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = x[v];
    if (!p.sigmoid) {
        float mx = x[0];
#pragma unroll
        for (int v = 1; v < V; ++v) mx = fmaxf(mx, x[v]);
        mx = row_max(mx);
        odd |= mx == INFINITY;
        if (scored) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                c[v] = x[v] == none ? 0.0f : __expf(x[v] - mx);
                sum += c[v];
            }
            const float inv = __builtin_amdgcn_rcpf(row_sum(sum));
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = x[v] == none ? none : c[v] * inv;
            err = inv * (0x1p-23f * (13.0f + V / 2));
        }
    } else if (scored) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            c[v] = x[v] == none ? none : __builtin_amdgcn_rcpf(1.0f + __expf(-x[v]));
        err = 0x1p-22f;
    }
    if (p.bias) {  // (-inf stays, unless the bias is infinite or a NaN: then the row is odd)
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] += b[v];
    }
    float mx = none;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        odd |= c[v] != c[v];
        mx = fmaxf(mx, c[v]);
    }
    mx = row_max(mx);
    odd |= mx == INFINITY;
    bool ok = true, open = true;
    if (G) {
        open = group_stays<V>(p, c, l / lanes, err, ok);
        ok = ok || !scored;  // (the largest logits themselves: equal ones go by the index)
    }
    if (scored) err += 0x1p-23f * fabsf(mx);
    if (!p.bias) {  // the experts by their logits
        mx = none;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            c[v] = x[v];
            mx = fmaxf(mx, open ? c[v] : none);
        }
        mx = row_max(mx);
    }
    const bool keyed = p.bias != nullptr;
    uint32_t key[V];
    uint32_t apart = 1;  // by how much fixed-point neighbours have to differ
    constexpr bool kExact = DT == NSOSX_BF16;
    const bool exact = kExact && !keyed;
    if (exact) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            // (adding +0 turns -0 into +0: equal values make equal keys)
            const uint32_t u = __float_as_uint(c[v] + 0.0f) >> 16;
            const uint32_t o = u & 0x8000u ? ~u & 0xFFFFu : u | 0x8000u;
            key[v] = open && c[v] != none ? (o << 16) | (0xFFFFu - (first + v * step)) : 0u;
        }
    } else {
        const float scale = keyed ? (float)(1u << (NB - 1)) : (float)(1u << (NB - 5));
        const float base = mx - (keyed ? 2.0f : 32.0f);
        const float top = (float)(1u << NB) - (NB > 24 ? (float)(1u << (NB - 24)) : 1.0f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            // (nothing available, -inf, lies below the window, whose keys are never trusted; an index
            // past the last expert's is one of those)
            const float t = fminf(fmaxf(((open ? c[v] : none) - base) * scale, 0.0f), top);
            key[v] = ((uint32_t)t << IB) | ((kIndex - (first + v * step)) & kIndex);
        }
        // both values' errors, the difference's and the product's rounding, the truncation
        if (keyed) apart = (uint32_t)fminf(2.0f * err * scale, 1e9f) + (1u << (NB > 24 ? NB - 23 : 1)) + 2;
    }
    sort_keys<0, V>(key);
    uint32_t mine = 0, before = 0;  // lane l's: the key of choice l, and of the one behind the last
    bool inside = true, clear = true;
    auto next = [&](int i) {  // the row's largest key, out of its lane's list
        const uint32_t m = row_max(key[0]);
        clear = clear && (exact || i == 0 || (before >> IB) >= (m >> IB) + apart);
        before = m;
        if (l == i) mine = m;
        if (key[0] == m) {  // (as selects, the compiler made this a search through the array)
#pragma unroll
            for (int v = 0; v + 1 < V; ++v) key[v] = key[v + 1];
            key[V - 1] = 0;
        }
        return m;
    };
    for (int i = 0; i < p.k; ++i) {
        const uint32_t m = next(i);
        inside = inside && (exact || (m >> IB) != 0);
    }
    next(p.k);  // (it only has to be apart from the last choice)
    odd = row_any(odd);
    sure = !live || (ok && inside && clear && !odd);
    int choice = exact ? (int)(0xFFFFu - (mine & 0xFFFFu)) : (int)(kIndex - (mine & kIndex));
    if (l >= p.k || mine == 0) choice = -1;
    // Only choices too close to each other: where the k + 1 largest are apart from all others, they are
    // put in order in 64 bits, one a lane.
    const bool close = live && ok && inside && !clear && !odd && !exact && p.k < 16 && (!p.bias || p.sigmoid);
    if (__any(close)) {
        const uint32_t m = row_max(key[0]);
        const bool settled = close && (before >> IB) >= (m >> IB) + apart;
        const int e = min((int)(kIndex - (mine & kIndex)), p.E - 1);
        double val = (double)load_act<DT>(p.logits, row * p.stride + e);
        if (p.bias) val = 1.0 / (1.0 + exp_of(-val)) + (double)p.bias[e];
        if (l > p.k || mine == 0) val = -(double)INFINITY;
        int rank = 0;
        outranked64<1>(val, e, rank); outranked64<2>(val, e, rank); outranked64<3>(val, e, rank);
        outranked64<4>(val, e, rank); outranked64<5>(val, e, rank); outranked64<6>(val, e, rank);
        outranked64<7>(val, e, rank); outranked64<8>(val, e, rank); outranked64<9>(val, e, rank);
        outranked64<10>(val, e, rank); outranked64<11>(val, e, rank); outranked64<12>(val, e, rank);
        outranked64<13>(val, e, rank); outranked64<14>(val, e, rank); outranked64<15>(val, e, rank);
        const uint32_t at = (uint32_t)(l > p.k ? 16 : rank) << 16 | (uint32_t)e;
        uint32_t got = at;
        ranked_here<1>(at, l, got); ranked_here<2>(at, l, got); ranked_here<3>(at, l, got);
        ranked_here<4>(at, l, got); ranked_here<5>(at, l, got); ranked_here<6>(at, l, got);
        ranked_here<7>(at, l, got); ranked_here<8>(at, l, got); ranked_here<9>(at, l, got);
        ranked_here<10>(at, l, got); ranked_here<11>(at, l, got); ranked_here<12>(at, l, got);
        ranked_here<13>(at, l, got); ranked_here<14>(at, l, got); ranked_here<15>(at, l, got);
        if (settled) {
            sure = true;
            choice = l < p.k ? (int)(got & 0xFFFFu) : -1;
        }
    }
    return live ? choice : -1;
}

// Step O of a reduction over a wave: a rotation within the 16-lane rows for 1 .. 8, the rows
// exchanged for 16 and 32.
template <int O>
__device__ __forceinline__ uint32_t wave_move(uint32_t v) {
    if constexpr (O < 16) {
        return ror16<O>(v);
    } else if constexpr (O == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? p[0] : p[1];
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? p[0] : p[1];
    }
}
template <int O>
__device__ __forceinline__ double wave_move(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = wave_move<O>((uint32_t)u), hi = wave_move<O>((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, lo | (hi << 32));
}
template <int O = 32>
__device__ __forceinline__ double wave_max(double v) {
    v = fmax(v, wave_move<O>(v));
    if constexpr (O > 1) v = wave_max<O / 2>(v);
    return v;
}
template <int O = 32>
__device__ __forceinline__ double wave_sum(double v) {
    v += wave_move<O>(v);
    if constexpr (O > 1) v = wave_sum<O / 2>(v);
    return v;
}
template <int O = 32>
__device__ __forceinline__ void wave_max2(double& a, double& b) {
    const double oa = wave_move<O>(a), ob = wave_move<O>(b);
    b = fmax(fmin(a, oa), fmax(b, ob));
    a = fmax(a, oa);
    if constexpr (O > 1) wave_max2<O / 2>(a, b);
}
template <int CTRL>
__device__ __forceinline__ double dpp_move(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, lo | (hi << 32));
}
// The two largest of a and b here and in another lane.
__device__ __forceinline__ void join_two(double& a, double& b, double oa, double ob) {
    b = fmax(fmin(a, oa), fmax(b, ob));
    a = fmax(a, oa);
}
__device__ __forceinline__ double lane_value(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __builtin_bit_cast(double, lo | (hi << 32));
}

// One row (the same in every lane) chosen by a whole wave in 64 bits: choice i in every lane whose
// number mod 16 is i (-1 where no expert is left).  bad: the row holds a NaN, or an infinite logit
// that its softmax cannot take.  A lane has a run of experts, sorted, so that a round looks at one
// value a lane, and ties go to the lowest lane; groups (G) lie on lanes of their own.  One wave does
// this while the rest of its launch has ended, so every instruction shows (256 experts of 8 groups: 4
// us, and 8 with the experts strewn over the lanes and a wave's reduction for each group).
template <int V, int DT, bool G>
__device__ __forceinline__ int select_wave(const RouteScored& p, int64_t row, bool& bad) {
    constexpr int W = V > 4 ? V / 4 : 1;
    const double none = -(double)INFINITY;
    const int lane = threadIdx.x & 63;
    const bool scored = p.bias || (G && p.best == 2);
    const bool apart = G && (V < 32 || p.lanes > 0);  // groups on lanes of their own
    const int lanes = apart ? 4 * p.lanes : 64;  // (a power of two)
    const int q = lane / lanes, all = apart ? p.size : p.E;
    const int run = (all + lanes - 1) / lanes, at = (lane & (lanes - 1)) * run;
    const int first = q * all + at, n = q * all < p.E ? min(run, all - at) : 0;
    float x[W];
    double c[W];
    int expert[W];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < W; ++v) {
        expert[v] = min(first + v, p.E - 1);
        x[v] = load_act<DT>(p.logits, row * p.stride + expert[v]);
        x[v] = v < n ? x[v] : -INFINITY;
        nan |= x[v] != x[v];
        c[v] = (double)x[v];
    }
    if (p.sigmoid) {
        if (scored) {
#pragma unroll
            for (int v = 0; v < W; ++v)
                c[v] = c[v] > none ? 1.0 / (1.0 + exp_of(-c[v])) : c[v];
        }
    } else {
        double mx = c[0], sum = 0.0;
#pragma unroll
        for (int v = 1; v < W; ++v) mx = fmax(mx, c[v]);
        mx = wave_max(mx);
        nan |= mx == (double)INFINITY;
        if (scored) {
#pragma unroll
            for (int v = 0; v < W; ++v) {
                c[v] = c[v] > none ? exp_of(c[v] - mx) : c[v];
                sum += c[v] > none ? c[v] : 0.0;
            }
            sum = wave_sum(sum);
#pragma unroll
            for (int v = 0; v < W; ++v) c[v] = c[v] > none ? c[v] / sum : c[v];
        }
    }
    if (p.bias) {
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const double b = (double)p.bias[expert[v]];
            c[v] = c[v] > none ? c[v] + b : c[v];
            nan |= c[v] != c[v];
        }
    }
    bad = __any(nan);
    if (apart) {
        double a = none, b = none;  // the group's two largest
#pragma unroll
        for (int v = 0; v < W; ++v) {
            b = fmax(b, fmin(a, c[v]));
            a = fmax(a, c[v]);
        }
        join_two(a, b, dpp_move<0xB1>(a), dpp_move<0xB1>(b));  // lane l ^ 1
        join_two(a, b, dpp_move<0x4E>(a), dpp_move<0x4E>(b));  // lane l ^ 2
        if (lanes >= 8) join_two(a, b, dpp_move<0x141>(a), dpp_move<0x141>(b));  // l ^ 7: the other four
        if (lanes >= 16) join_two(a, b, dpp_move<0x140>(a), dpp_move<0x140>(b));  // l ^ 15: the other eight
        if (lanes >= 32) join_two(a, b, wave_move<16>(a), wave_move<16>(b));
        const double s = p.best == 2 && b > none ? a + b : a;
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double o = lane_value(s, g * lanes);
            rank += o > s || (o == s && g < q) ? 1 : 0;
        }
        const bool open = rank < p.keep;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            if (!p.bias) c[v] = (double)x[v];  // the experts by their logits
            c[v] = open && v < n ? c[v] : none;
        }
    } else if constexpr (G && V == 32) {
        double s = none;  // lane g's: the score of group g
        for (int g = 0; g < p.groups; ++g) {
            double a = none, b = none;
#pragma unroll
            for (int v = 0; v < W; ++v) {
                const int e = first + v;
                const double u = e >= g * p.size && e < (g + 1) * p.size ? c[v] : none;
                b = fmax(b, fmin(a, u));
                a = fmax(a, u);
            }
            wave_max2(a, b);
            if (lane == g) s = p.best == 2 && b > none ? a + b : a;
        }
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            const double o = lane_value(s, g);
            rank += o > s || (o == s && g < lane) ? 1 : 0;
        }
        const uint64_t kept = __ballot(lane < p.groups && rank < p.keep);
#pragma unroll
        for (int v = 0; v < W; ++v) {
            if (!p.bias) c[v] = (double)x[v];
            if (!((kept >> (expert[v] / p.size)) & 1)) c[v] = none;
        }
    }
    // (neighbours change places only where the first is smaller: equal values stay in order)
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int v = i & 1; v + 1 < W; v += 2) {
            const bool swap = c[v] < c[v + 1];
            const double hi = swap ? c[v + 1] : c[v], lo = swap ? c[v] : c[v + 1];
            const int eh = swap ? expert[v + 1] : expert[v], el = swap ? expert[v] : expert[v + 1];
            c[v] = hi;
            c[v + 1] = lo;
            expert[v] = eh;
            expert[v + 1] = el;
        }
    int mine = -1;
    for (int i = 0; i < p.k; ++i) {
        const double top = wave_max(c[0]);
        const uint64_t holders = __ballot(c[0] == top);
        const int holder = holders ? __builtin_ctzll(holders) : 0;
        const int e = top > none ? __builtin_amdgcn_readlane(expert[0], holder) : -1;
        if (lane == holder) {
#pragma unroll
            for (int v = 0; v + 1 < W; ++v) {
                c[v] = c[v + 1];
                expert[v] = expert[v + 1];
            }
            c[W - 1] = none;
        }
        if ((lane & 15) == i) mine = e;
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
            row_values<V, DT>(p.logits, row * p.stride, p.E, live, all);
            softmax_stats<V>(all, mx, sum);
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

// Inclusive scan over a wave.
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int u = __shfl_up(v, o, kWave);
        if (lane >= o) v += u;
    }
    return v;
}

// Exclusive scan of counts [E] into s_off [E + 1] by the first wave of a workgroup: each lane
// takes a run of 8, all loads at once.
__device__ __forceinline__ void scan_counts(const int32_t* counts, int E, int32_t* s_off) {
    if (threadIdx.x >= kWave) return;
    const int first = threadIdx.x * 8;
    int c[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = first + i < E ? counts[first + i] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += c[i];
    int at = wave_scan(sum) - sum;
    static_assert(kScoredMaxExperts == 8 * kWave, "a wave's runs hold every expert");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (first + i <= E) s_off[first + i] = at;
        at += c[i];
    }
    if (E == kScoredMaxExperts && threadIdx.x == kWave - 1) s_off[E] = at;
}

// A workgroup of 16 RB threads routes RB rows, ranks them per expert through 64-bit row masks
// and leaves its counts per expert, or, where it is the only one, the whole dispatch.
template <int V, int DT, bool G>
__global__ __launch_bounds__(V > 16 ? 512 : 1024) void route_scored_kernel(RouteScored p) {
    __shared__ uint64_t s_mask[kScoredMaxExperts];
    __shared__ int32_t s_cnt[kScoredMaxExperts], s_off[kScoredMaxExperts + 1];
    const int l = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int row = blockIdx.x * (blockDim.x >> 4) + rl;
    extern __shared__ __align__(16) float s_rows[];  // G: a row each, and the biases
    float* s_bias = s_rows + (blockDim.x >> 4) * p.pitch;
    const bool dispatch = p.counts != nullptr;
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
        if (dispatch) s_mask[e] = 0;
        if (G && p.bias) s_bias[e] = p.bias[e];
    }
    __syncthreads();
    const int in = min(row, p.rows - 1);  // a row to read, past the last one too
    const bool live = row < p.rows && (!p.valid || p.valid[in] != 0);
    bool bad = false, sure;
    int mine = select_fast<V, DT, G>(p, in, live, s_rows + rl * p.pitch, s_bias, sure);
    if (G && p.lanes == 0) sure = !live;  // groups that the lanes cannot hold
    for (uint64_t left = __ballot(!sure && l == 0); left; left &= left - 1) {
        const int first = __builtin_ctzll(left);
        bool wrong;
        const int c = select_wave<V, DT, G>(p, __builtin_amdgcn_readlane(in, first), wrong);
        if ((int)(threadIdx.x & 48) == first) {
            mine = c;
            bad = wrong;
        }
    }
    if (live && bad) mine = l < p.k ? l : -1;  // a NaN score: the first k experts, weights NaN
    float w = row_weight<V, DT>(p, in, live, mine);
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
        if (p.by_block) {
            const int words = (p.E + 3) / 4;
            for (int i = threadIdx.x; i < words; i += blockDim.x) {
                uint32_t w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * i + j < p.E) w |= (uint32_t)__popcll(s_mask[4 * i + j]) << (8 * j);
                p.block_counts[blockIdx.x * words + i] = (int32_t)w;
            }
        } else {
            for (int e = threadIdx.x; e < p.E; e += blockDim.x)
                p.block_counts[(int64_t)e * gridDim.x + blockIdx.x] = __popcll(s_mask[e]);
        }
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

// Per expert (a wave each): the exclusive scan of its counts over the blocks, in place, 256 blocks
// at a time.
__global__ __launch_bounds__(256) void route_scored_scan_kernel(int32_t* __restrict__ block_counts,
                                                                int blocks, int E,
                                                                int32_t* __restrict__ counts) {
    const int e = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (e >= E) return;
    const int lane = threadIdx.x & 63;
    int32_t* row = block_counts + (int64_t)e * blocks;
    int carry = 0;
    for (int b0 = 0; b0 < blocks; b0 += 4 * kWave) {
        const int b = b0 + 4 * lane;
        int c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = b + i < blocks ? row[b + i] : 0;
        const int sum = c[0] + c[1] + c[2] + c[3];
        const int upto = wave_scan(sum);
        int at = carry + upto - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (b + i < blocks) row[b + i] = at;
            at += c[i];
        }
        carry += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (lane == 0) counts[e] = carry;
}

// Ranks within a block -> slots.
__device__ __forceinline__ void place_entry(const RouteScored& p, const int32_t* s_off, int64_t i,
                                            int row, int e, int rank) {
    if (e >= 0) {
        p.slot_of[i] = s_off[e] + rank;
        p.perm[s_off[e] + rank] = row;
    }
    if (i >= s_off[p.E]) p.perm[i] = -1;
}

__global__ __launch_bounds__(256) void route_scored_place_kernel(RouteScored p, int blocks,
                                                                 int block_rows) {
    __shared__ int32_t s_off[kScoredMaxExperts + 1];
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const bool entry = i < (int64_t)p.rows * p.k;
    const int row = entry ? (int)(i / p.k) : 0, e = entry ? p.selected[i] : -1;
    const int rank =
        e >= 0 ? p.block_counts[(int64_t)e * blocks + row / block_rows] + p.slot_of[i] : -1;
    scan_counts(p.counts, p.E, s_off);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int j = threadIdx.x; j <= p.E; j += blockDim.x) p.offsets[j] = s_off[j];
    if (entry) place_entry(p, s_off, i, row, e, rank);
}

// The same with the scans over the blocks, for few counts (kScoredPlaceWords): a workgroup for each
// block of rows, which sums every expert's counts, and those before its own block, by itself.  A
// block has at most 64 rows, so its counts are bytes, four experts a word, summed in pairs of 16
// bits (an expert's count is at most the rows, below 65536); a thread loads its words (16, a few
// more at some widths) 16 at once, without a branch, and places one entry.  4096 rows of 60 experts: 4.8 us behind the selection, 16384 of 256
// 6.8, where the two launches took 5.7 (their counts summed in one) and 7.7.
constexpr int kScoredPlaceThreads = 1024, kScoredPlaceWords = 16 * kScoredPlaceThreads;

__global__ __launch_bounds__(kScoredPlaceThreads) void route_scored_scan_place_kernel(RouteScored p,
                                                                                      int blocks,
                                                                                      int block_rows) {
    static_assert(kScoredMaxK * 64 <= kScoredPlaceThreads, "a thread an entry");
    __shared__ uint32_t s_sum[4][kScoredMaxExperts / 4];  // even and odd bytes: all, before this block
    __shared__ int32_t s_all[kScoredMaxExperts], s_before[kScoredMaxExperts], s_off[kScoredMaxExperts + 1];
    const int tid = threadIdx.x;
    const int64_t i = (int64_t)blockIdx.x * block_rows * p.k + tid;
    const bool entry = tid < block_rows * p.k && i < (int64_t)p.rows * p.k;
    const int e = entry ? p.selected[i] : -1, rank = entry ? p.slot_of[i] : 0;
    const int words = (p.E + 3) / 4, parts = min(kScoredPlaceThreads / words, (blocks + 15) / 16);
    if (tid < kScoredMaxExperts) (&s_sum[0][0])[tid] = 0;
    __syncthreads();
    const int part = tid / words, w = tid - part * words;
    if (part < parts) {
        const uint32_t* column = reinterpret_cast<const uint32_t*>(p.block_counts) + w;
        const int b0 = blocks * part / parts, b1 = blocks * (part + 1) / parts;
        uint32_t even = 0, odd = 0, even_before = 0, odd_before = 0;
        for (int first = b0; first < b1; first += 16) {  // (once or twice; loads past the end are clamped)
            uint32_t c[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) c[j] = column[min(first + j, b1 - 1) * words];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int b = first + j;
                const uint32_t lo = b < b1 ? c[j] & 0x00FF00FFu : 0, hi = b < b1 ? (c[j] >> 8) & 0x00FF00FFu : 0;
                even += lo;
                odd += hi;
                even_before += b < (int)blockIdx.x ? lo : 0;
                odd_before += b < (int)blockIdx.x ? hi : 0;
            }
        }
        atomicAdd(&s_sum[0][w], even);  // (whole numbers: in any order)
        atomicAdd(&s_sum[1][w], odd);
        atomicAdd(&s_sum[2][w], even_before);
        atomicAdd(&s_sum[3][w], odd_before);
    }
    __syncthreads();
    if (tid < p.E) {
        const int shift = tid & 2 ? 16 : 0;
        s_all[tid] = (s_sum[tid & 1][tid >> 2] >> shift) & 0xFFFF;
        s_before[tid] = (s_sum[2 + (tid & 1)][tid >> 2] >> shift) & 0xFFFF;
    }
    __syncthreads();
    scan_counts(s_all, p.E, s_off);
    __syncthreads();
    if (blockIdx.x == 0) {
        if (tid <= p.E) p.offsets[tid] = s_off[tid];
        if (tid < p.E) p.counts[tid] = s_all[tid];
    }
    if (entry) place_entry(p, s_off, i, (int)(i / p.k), e, e >= 0 ? s_before[e] + rank : -1);
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

// Whether another choice of the row, N lanes on, names the same expert (N up to 8 meets every pair).
template <int N>
__device__ __forceinline__ void same_expert(int e, bool& twice) {
    twice |= e >= 0 && ror16<N>(e) == e;
}

template <int V, int DT>
__global__ __launch_bounds__(256) void route_scored_bwd_kernel(RouteScoredBwd p) {
    extern __shared__ __align__(16) float s_g[];  // [16, E]
    const int l = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int row = blockIdx.x * 16 + rl;
    const bool live = row < p.rows;
    for (int i = threadIdx.x; i < 4 * p.E; i += 256)
        reinterpret_cast<float4*>(s_g)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    const int64_t base = (int64_t)min(row, p.rows - 1) * p.stride;
    const int64_t at = (int64_t)row * p.k + l;
    int e = live && l < p.k ? p.selected[at] : -1;
    if (e >= p.E) e = -1;
    const float none = -INFINITY;
    const float x = e >= 0 ? load_act<DT>(p.logits, base + e) : none;
    float g = e >= 0 ? p.dweights[at] * p.scale : 0.0f;
    const bool dense = !p.renorm && !p.sigmoid;
    float mx = none, sum = 1.0f, dot = 0.0f;
    float all[V];
    const bool chosen = row_any(e >= 0);  // a row without a choice, padding's, may hold anything
    if (dense) {
        row_values<V, DT>(p.logits, base, p.E, live, all);
        softmax_stats<V>(all, mx, sum);
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
    // An expert named twice gets both, one lane after the other (the order is the same each time); a
    // wave without one, every routing's, stores at once.
    bool twice = false;
    same_expert<1>(e, twice); same_expert<2>(e, twice); same_expert<3>(e, twice); same_expert<4>(e, twice);
    same_expert<5>(e, twice); same_expert<6>(e, twice); same_expert<7>(e, twice); same_expert<8>(e, twice);
    if (__any(twice)) {
        for (int i = 0; i < p.k; ++i)
            if (l == i && e >= 0) s_g[rl * p.E + e] += g;
    } else if (e >= 0) {
        s_g[rl * p.E + e] = g;
    }
    if (dense) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = 16 * v + l;
            if (j < p.E) {
                const float d = s_g[rl * p.E + j];
                s_g[rl * p.E + j] =
                    !chosen || all[v] == none ? 0.0f : (expf(all[v] - mx) / sum) * (d - dot);
            }
        }
    }
    __syncthreads();
    // the workgroup's rows lie behind each other: out in 16-byte pieces
    const int64_t first = (int64_t)blockIdx.x * 16 * p.E;
    const int count = min(16, p.rows - (int)blockIdx.x * 16) * p.E;
    constexpr int kPiece = DT == NSOSX_F32 ? 4 : 8;
    const int pieces = (reinterpret_cast<uintptr_t>(p.dlogits) & 15) == 0 ? count / kPiece : 0;
    for (int i = threadIdx.x; i < pieces; i += 256) {
        const float4 a = *reinterpret_cast<const float4*>(s_g + i * kPiece);
        if constexpr (DT == NSOSX_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p.dlogits) + first + i * kPiece) = a;
        } else {
            const float4 b = *reinterpret_cast<const float4*>(s_g + i * kPiece + 4);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dlogits) + first + i * kPiece) =
                make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                           pack_bf16x2(b.z, b.w));
        }
    }
    for (int i = pieces * kPiece + threadIdx.x; i < count; i += 256)
        store_act<DT>(p.dlogits, first + i, s_g[i]);
}

// Lanes of each group and values of a lane where G groups of `size` experts share 16 lanes.
struct ScoredLayout {
    int lanes, values;
};
static ScoredLayout scored_layout(int E, int groups) {
    int lanes = 16;
    while (lanes * groups > 16) lanes /= 2;
    return {lanes, (E / groups + lanes - 1) / lanes};
}

// wide: lanes of 32 values, whose kernel has the registers of half as many threads.
static int scored_block_rows(int rows, bool wide) {
    if (rows <= 16) return 16;
    if (rows <= 32) return 32;
    const int most = wide ? 32 : 64;
    if (rows <= 64) return most;
    return rows <= 4096 ? 16 : rows <= 8192 ? 32 : most;
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int64_t nsosx_moe_route_scored_workspace(int rows, int experts) {
    if (rows <= 0 || experts <= 0 || experts > kScoredMaxExperts) return 0;
    const int rb = scored_block_rows(rows, experts > 128);  // (128 or less are never wide)
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
    if ((int64_t)rows * k > 2147483647LL || rows > kScoredMaxRows)
        return fail(NSOSX_ERR_OVERFLOW, "moe_route_scored: rows*k or rows too large");
    const int limited = group_keep == groups ? 1 : groups;
    ScoredLayout at = scored_layout(experts, limited);
    // more experts of a group than its lanes hold (more than 288 in 9 .. 15 groups, say): every row is
    // chosen by a wave
    const bool spread = at.values <= 32;
    if (!spread) at = {0, 32};
    // without the dispatch a row needs no other: the smallest blocks (64 rows of 256 experts on one CU
    // 12 us, on four 7)
    const int rb = select_only ? 16 : scored_block_rows(rows, at.values > 16);
    const int blocks = (rows - 1) / rb + 1;
    const RouteScored p{logits, logits_stride, valid_rows, bias, rows, experts, k, sigmoid != 0, limited,
                        group_keep, group_best, renorm != 0, scale, weights, selected, counts, offsets,
                        perm, slot_of, workspace,
                        rows <= 65535 && (int64_t)blocks * ((experts + 3) / 4) <= kScoredPlaceWords,
                        experts / limited, at.lanes, at.values,
                        (experts + 63) / 64 * 64 + 16};  // (four rows' lanes on different banks)
    const int smem = limited > 1 ? (rb * p.pitch + (experts + 3) / 4 * 4) * 4 : 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define NSOSX_RS_DT(V, G)                                                                       \
    if (logits_dtype == NSOSX_F32)                                                              \
        hipLaunchKernelGGL((route_scored_kernel<V, NSOSX_F32, G>), dim3(blocks), dim3(16 * rb), \
                           smem, st, p);                                                        \
    else                                                                                        \
        hipLaunchKernelGGL((route_scored_kernel<V, NSOSX_BF16, G>), dim3(blocks), dim3(16 * rb), \
                           smem, st, p);
#define NSOSX_RS(V)                                                    \
    do {                                                               \
        if (p.groups > 1) { NSOSX_RS_DT(V, true) } else { NSOSX_RS_DT(V, false) } \
    } while (0)
    NSOSX_SCORED_V(16 * at.values, NSOSX_RS);
#undef NSOSX_RS_DT
#undef NSOSX_RS
    if (!select_only && blocks > 1 && p.by_block) {
        hipLaunchKernelGGL(route_scored_scan_place_kernel, dim3(blocks), dim3(kScoredPlaceThreads), 0, st, p,
                           blocks, rb);
    } else if (!select_only && blocks > 1) {
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
    if ((int64_t)rows * k > 2147483647LL || rows > kScoredMaxRows)
        return fail(NSOSX_ERR_OVERFLOW, "moe_route_scored_backward: rows*k or rows too large");
    const int64_t size = logits_dtype == NSOSX_F32 ? 4 : 2, db = (int64_t)rows * experts * size;
    if (overlaps(dlogits, db, logits, ((int64_t)(rows - 1) * logits_stride + experts) * size) ||
        overlaps(dlogits, db, selected, (int64_t)rows * k * 4) ||
        overlaps(dlogits, db, dweights, (int64_t)rows * k * 4))
        return fail(NSOSX_ERR_INVALID, "moe_route_scored_backward: dlogits overlaps an input");
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
