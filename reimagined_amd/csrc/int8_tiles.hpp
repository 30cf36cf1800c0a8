// Tiles of the int8 x int8 products (int8_gemm.hip): the few-row tile, whose waves split K,
// and the LDS-staged block tile.
#pragma once
#include "common.hpp"

namespace nsosx {

typedef int i8x16 __attribute__((ext_vector_type(4)));   // 16 int8 operand bytes of a lane
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kI8MaxK = 131071;       // 128 * 128 * K stays in int32
constexpr int kI8MaxExperts = 1024;

// Weights [N, K] with a scale (and an optional bias) per output.
struct I8Problem {
    const int8_t* w;
    const float* w_scale;
    const float* bias;
    int N, K;
    int sqrelu;
};

// Rows begin .. begin + count of the output; output row r reads row perm[r] (r itself where
// perm is null) of the q_rows rows of q.
struct I8Rows {
    const int8_t* q;
    const float* act_scale;
    const int32_t* perm;
    int begin, count;
    int q_rows;
};

struct I8Group {
    const int8_t* w;          // [experts, N, K]
    const float* w_scale;     // [experts, N]
    const float* bias;        // [experts, N] or null
    const int8_t* q;
    const float* act_scale;
    const int32_t* offsets;   // [experts + 1]
    const int32_t* perm;
    int q_rows, slots, experts, N, K;
    int sqrelu;
};

// The row of q behind output row r; an index outside q (no routing makes one) is clamped, so
// that it reads a wrong row and not past the buffer.
__device__ __forceinline__ int i8_source(const I8Rows& rows, int r) {
    const int s = rows.perm ? rows.perm[r] : r;
    return min(max(s, 0), rows.q_rows - 1);
}

__device__ __forceinline__ bool i8_segment(const I8Group& gp, int e, I8Problem& pb, I8Rows& rows) {
    const int b = min(max(gp.offsets[e], 0), gp.slots);
    const int n = min(max(gp.offsets[e + 1], 0), gp.slots) - b;
    if (n <= 0) return false;
    const int64_t o = (int64_t)e * gp.N;
    pb = I8Problem{gp.w + o * gp.K, gp.w_scale + o, gp.bias ? gp.bias + o : nullptr, gp.N, gp.K,
                   gp.sqrelu};
    rows = I8Rows{gp.q, gp.act_scale, gp.perm, b, n, gp.q_rows};
    return true;
}

// Row tile `tile` of the experts' segments in order (ceil(rows / BM) tiles each): its expert
// and first row.  A wave counts 64 experts' tiles at a time.
template <int BM>
__device__ __forceinline__ bool i8_find_segment(const I8Group& gp, int tile, int& e, int& m0) {
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < gp.experts; e0 += kWave) {
        const int j = e0 + lane;
        int tiles = 0;
        if (j < gp.experts) {
            const int b = min(max(gp.offsets[j], 0), gp.slots);
            const int n = min(max(gp.offsets[j + 1], 0), gp.slots) - b;
            tiles = n > 0 ? (n + BM - 1) / BM : 0;
        }
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int v = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += v;
        }
        const uint64_t past = __ballot(tile < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            e = e0 + l;
            m0 = (tile - __builtin_amdgcn_readlane(upto - tiles, l)) * BM;
            return true;
        }
        tile -= __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return false;
}

// 16 bytes at any address (a row starts at any byte where K is no multiple of 16).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ i8x16 load16(const int8_t* p) {
    const u32x4_any v = *(const __attribute__((address_space(1))) u32x4_any*)(p);
    return i8x16{(int)v.x, (int)v.y, (int)v.z, (int)v.w};
}

// Bytes k .. k + 15 of a row, zeros past K.
__device__ __forceinline__ i8x16 load16_tail(const int8_t* row, int k, int K) {
    if (k + 16 <= K) return load16(row + k);
    uint32_t d[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < K) d[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    return i8x16{(int)d[0], (int)d[1], (int)d[2], (int)d[3]};
}

// The affine of one output.  Rounded at the conversion, both products and the sum.
__device__ __forceinline__ float i8_affine(int acc, float as, float ws, float bias, int sqrelu) {
    float v = __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(acc), as), ws), bias);
    if (sqrelu) {
        v = v < 0.0f ? 0.0f : v;  // a NaN stays
        v = __fmul_rn(v, v);
    }
    return v;
}

// ===========================================================================
// Few rows: a workgroup owns 16 outputs x 16 MT tokens and its eight waves split K.  Every
// wave runs v_mfma_i32_16x16x64_i8 on fragments straight from memory (lane l: row l % 16, the
// 16 bytes of K quarter l / 16), so a 64-deep step reads 64 contiguous bytes of 16 weight
// rows; the partial sums meet in LDS.  What bounds it is the read of the weights.
// ===========================================================================
constexpr int kSkinnyWaves = 8;
constexpr int kSkinnyThreads = 64 * kSkinnyWaves;

constexpr int i8_skinny_smem(int mt) { return kSkinnyWaves * mt * 256 * 4; }

template <int YDT, int MT>
__device__ __forceinline__ void i8_skinny_tile(const I8Problem& pb, const I8Rows& rows, int n0,
                                               int m0, void* __restrict__ y,
                                               int32_t* __restrict__ s_part) {
    constexpr int U = MT >= 4 ? 4 : 8;  // steps whose loads are in flight together
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    // rows past N or the segment re-read its last one; their outputs are not stored
    const int8_t* wrow = pb.w + (int64_t)min(n0 + r, pb.N - 1) * pb.K + 16 * g;
    const int8_t* xrow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        xrow[t] = rows.q + (int64_t)i8_source(rows, rows.begin + min(m0 + 16 * t + r, rows.count - 1)) *
                               pb.K + 16 * g;
    i8x16 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = i8x16{0, 0, 0, 0};
    const int steps = pb.K / 64;
    const int s0 = steps * wave / kSkinnyWaves, s1 = steps * (wave + 1) / kSkinnyWaves;
    int s = s0;
    for (; s + U <= s1; s += U) {
        i8x16 a[U], b[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            a[u] = load16(wrow + (int64_t)(s + u) * 64);
#pragma unroll
            for (int t = 0; t < MT; ++t) b[u][t] = load16(xrow[t] + (int64_t)(s + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u][t], acc[t], 0, 0, 0);
    }
    for (; s < s1; ++s) {
        const i8x16 a = load16(wrow + (int64_t)s * 64);
#pragma unroll
        for (int t = 0; t < MT; ++t)
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, load16(xrow[t] + (int64_t)s * 64),
                                                           acc[t], 0, 0, 0);
    }
    if (wave == kSkinnyWaves - 1 && steps * 64 < pb.K) {
        const int k = steps * 64 + 16 * g;
        const i8x16 a = load16_tail(wrow - 16 * g, k, pb.K);
#pragma unroll
        for (int t = 0; t < MT; ++t)
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                a, load16_tail(xrow[t] - 16 * g, k, pb.K), acc[t], 0, 0, 0);
    }
    // accumulator c of lane l: output n0 + 4 (l / 16) + c, token m0 + 16 t + l % 16
#pragma unroll
    for (int t = 0; t < MT; ++t)
        *reinterpret_cast<int4*>(s_part + ((wave * MT + t) * 64 + lane) * 4) =
            make_int4(acc[t].x, acc[t].y, acc[t].z, acc[t].w);
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * MT; i += kSkinnyThreads) {
        const int t = i >> 6, l = i & 63;
        const int m = m0 + 16 * t + (l & 15), n = n0 + 4 * (l >> 4);
        if (m >= rows.count || n >= pb.N) continue;
        int sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kSkinnyWaves; ++w) {
            const int4 v = *reinterpret_cast<const int4*>(s_part + ((w * MT + t) * 64 + l) * 4);
            sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
        }
        const int64_t orow = rows.begin + m;
        const float as = rows.act_scale[i8_source(rows, (int)orow)];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (n + c < pb.N)
                store_act<YDT>(y, orow * pb.N + n + c,
                               i8_affine(sum[c], as, pb.w_scale[n + c],
                                         pb.bias ? pb.bias[n + c] : 0.0f, pb.sqrelu));
    }
}

// ===========================================================================
// Block tile: 64 NWN outputs x 32 TM NWM tokens, NWN x NWM waves of 64 x 32 TM = 2 x TM tiles
// of v_mfma_i32_32x32x32_i8, over 128-deep stages double-buffered in LDS.  A stage is fetched
// into registers while the one before it is multiplied.  16-byte chunk c of row r sits in slot
// c ^ ((r / 2) % 8), so that the 16 rows that one clock of a ds_read_b128 serves lie in
// different banks.
// ===========================================================================
constexpr int kI8BK = 128;

template <int NWN, int NWM, int TM>
constexpr int i8_tile_smem() { return 2 * (64 * NWN + 32 * TM * NWM) * kI8BK; }

__device__ __forceinline__ void i8_tile_order(int L, int ntn, int ntm, int& nt, int& mt) {
    const int total = ntn * ntm, per = total / 8;
    const int t = L < per * 8 ? (L % 8) * per + L / 8 : L;
    nt = t % ntn;
    mt = t / ntn;
}

template <int YDT, int NWN, int NWM, int TM>
__device__ __forceinline__ void i8_epilogue(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                            void* __restrict__ y, char* smem,
                                            const i32x16 (&acc)[2][TM]) {
    constexpr int kThreads = 64 * NWN * NWM, kSize = YDT == NSOSX_F32 ? 4 : 2;
    constexpr int kRow = 64 * kSize, kSlice = 32 * kRow, kChunks = kRow / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wn = wave % NWN, wm = wave / NWN;
    const int g = lane >> 5, li = lane & 31;
    float* s_scale = reinterpret_cast<float*>(smem + NWN * NWM * kSlice);
    float* s_bias = s_scale + 64 * NWN;
    __syncthreads();  // every wave is done with the stages
    for (int i = tid; i < 64 * NWN; i += kThreads) {
        const int n = min(n0 + i, pb.N - 1);
        s_scale[i] = pb.w_scale[n];
        s_bias[i] = pb.bias ? pb.bias[n] : 0.0f;
    }
    __syncthreads();
    char* slice = smem + wave * kSlice;
    const int nw = n0 + 64 * wn;
    const bool whole = nw + 64 <= pb.N && pb.N % (16 / kSize) == 0 &&
                       (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int mt = m0 + 32 * (wm * TM + t);
        if (mt >= rows.count) break;
        const float as = rows.act_scale[i8_source(rows, rows.begin + min(mt + li, rows.count - 1))];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const int at = 32 * nb + 8 * q4 + 4 * g;  // of the wave's 64 outputs
                const float4 sc = *reinterpret_cast<const float4*>(s_scale + 64 * wn + at);
                const float4 bs = *reinterpret_cast<const float4*>(s_bias + 64 * wn + at);
                const i32x16& a = acc[nb][t];
                const float o0 = i8_affine(a[4 * q4], as, sc.x, bs.x, pb.sqrelu);
                const float o1 = i8_affine(a[4 * q4 + 1], as, sc.y, bs.y, pb.sqrelu);
                const float o2 = i8_affine(a[4 * q4 + 2], as, sc.z, bs.z, pb.sqrelu);
                const float o3 = i8_affine(a[4 * q4 + 3], as, sc.w, bs.w, pb.sqrelu);
                const int chunk = at * kSize / 16;
                char* dst = slice + li * kRow + ((chunk ^ (li & (kChunks - 1))) << 4);
                if constexpr (YDT == NSOSX_F32)
                    *reinterpret_cast<float4*>(dst) = make_float4(o0, o1, o2, o3);
                else
                    *reinterpret_cast<uint2*>(dst + 8 * g) =
                        make_uint2(pack_bf16x2(o0, o1), pack_bf16x2(o2, o3));
            }
        // the wave reads back what its own lanes wrote
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (whole) {
            const int c = lane & (kChunks - 1);
#pragma unroll
            for (int i = 0; i < 32 * kChunks / 64; ++i) {
                const int row = i * (64 / kChunks) + lane / kChunks;
                const u32x4 v = *reinterpret_cast<const u32x4*>(
                    slice + row * kRow + ((c ^ (row & (kChunks - 1))) << 4));
                if (mt + row < rows.count)
                    __builtin_nontemporal_store(
                        v, reinterpret_cast<u32x4*>(static_cast<char*>(y) +
                                                    ((int64_t)(rows.begin + mt + row) * pb.N + nw) * kSize +
                                                    16 * c));
            }
        } else {
            const int last = min(32, rows.count - mt);
            for (int row = 0; row < last; ++row) {
                const char* src = slice + row * kRow +
                                  ((((lane * kSize) / 16) ^ (row & (kChunks - 1))) << 4) +
                                  (lane * kSize) % 16;
                if (nw + lane < pb.N) {
                    const int64_t at = (int64_t)(rows.begin + mt + row) * pb.N + nw + lane;
                    if constexpr (YDT == NSOSX_F32)
                        static_cast<float*>(y)[at] = *reinterpret_cast<const float*>(src);
                    else
                        static_cast<uint16_t*>(y)[at] = *reinterpret_cast<const uint16_t*>(src);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next tile's writes
    }
}

template <int YDT, int NWN, int NWM, int TM>
__device__ __forceinline__ void i8_tile(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                        void* __restrict__ y, char* smem) {
    constexpr int kThreads = 64 * NWN * NWM, BN = 64 * NWN, BM = 32 * TM * NWM;
    constexpr int kStage = (BN + BM) * kI8BK, kLoads = (BN + BM) * 8 / kThreads;
    static_assert((BN + BM) * 8 % kThreads == 0 && BN * 8 % kThreads == 0, "whole loads");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wn = wave % NWN, wm = wave / NWN;
    const int g = lane >> 5, li = lane & 31;
    // chunk i of a thread: row (i kThreads + tid) / 8 of the stage (weights, then tokens)
    const int8_t* src[kLoads];
    int kof[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int row = (i * kThreads + tid) >> 3;
        kof[i] = ((tid & 7) ^ ((row >> 1) & 7)) * 16;
        // rows past N or the segment re-read its last one; their outputs are not stored
        src[i] = i * kThreads < BN * 8
                     ? pb.w + (int64_t)min(n0 + row, pb.N - 1) * pb.K
                     : rows.q + (int64_t)i8_source(rows, rows.begin + min(m0 + row - BN, rows.count - 1)) * pb.K;
    }
    i8x16 reg[kLoads];
    const int KT = (pb.K + kI8BK - 1) / kI8BK;
    auto fetch = [&](int kt) {
        if ((kt + 1) * kI8BK <= pb.K) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) reg[i] = load16(src[i] + kt * kI8BK + kof[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) reg[i] = load16_tail(src[i], kt * kI8BK + kof[i], pb.K);
        }
    };
    auto put = [&](int kt) {
        char* st = smem + (kt & 1) * kStage + tid * 16;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *reinterpret_cast<i8x16*>(st + i * kThreads * 16) = reg[i];
    };
    i32x16 acc[2][TM];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = i32x16{};
    fetch(0);
    put(0);
    if (KT > 1) fetch(1);
    __syncthreads();
    for (int kt = 0; kt < KT; ++kt) {
        const char* wl = smem + (kt & 1) * kStage + (64 * wn + li) * kI8BK;
        const char* xl = smem + (kt & 1) * kStage + (BN + 32 * TM * wm + li) * kI8BK;
        const int sw = (li >> 1) & 7;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int slot = ((2 * ks + g) ^ sw) * 16;
            i8x16 a[2], b[TM];
#pragma unroll
            for (int n = 0; n < 2; ++n)
                a[n] = *reinterpret_cast<const i8x16*>(wl + n * 32 * kI8BK + slot);
#pragma unroll
            for (int t = 0; t < TM; ++t)
                b[t] = *reinterpret_cast<const i8x16*>(xl + t * 32 * kI8BK + slot);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int t = 0; t < TM; ++t)
                    acc[n][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[n], b[t], acc[n][t], 0, 0, 0);
        }
        if (kt + 1 < KT) {
            put(kt + 1);
            if (kt + 2 < KT) fetch(kt + 2);
        }
        __syncthreads();
    }
    i8_epilogue<YDT, NWN, NWM, TM>(pb, rows, n0, m0, y, smem, acc);
}

}  // namespace nsosx
