// Tiles of the int8 x int8 products (int8_gemm.hip): the one for few tiles, whose waves split K,
// and the block tiles, through registers (any alignment) or straight into LDS.
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

// Row tiles of expert j's segment.
template <int BM>
__device__ __forceinline__ int i8_row_tiles(const I8Group& gp, int j) {
    if (j >= gp.experts) return 0;
    const int n = min(max(gp.offsets[j + 1], 0), gp.slots) - min(max(gp.offsets[j], 0), gp.slots);
    return n > 0 ? (n + BM - 1) / BM : 0;
}

__device__ __forceinline__ int i8_wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int u = __shfl_up(v, o, kWave);
        if (lane >= o) v += u;
    }
    return v;
}

// All segments' row tiles.
template <int BM>
__device__ __forceinline__ int i8_all_tiles(const I8Group& gp) {
    int total = 0;
    for (int e0 = 0; e0 < gp.experts; e0 += kWave)
        total += wave_sum_i32(i8_row_tiles<BM>(gp, e0 + (threadIdx.x & 63)));
    return __builtin_amdgcn_readfirstlane(total);
}

// Row tile `tile` of the segments in order: its expert and first row.  A wave counts 64 experts at
// a time.
template <int BM>
__device__ __forceinline__ bool i8_find_segment(const I8Group& gp, int tile, int& e, int& m0) {
    for (int e0 = 0; e0 < gp.experts; e0 += kWave) {
        const int tiles = i8_row_tiles<BM>(gp, e0 + (threadIdx.x & 63));
        const int upto = i8_wave_scan(tiles);
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

// 16 bytes at any address (a row starts at any byte where K is no multiple of 16).  The unit takes
// such loads as they are; the five words that hold them, loaded and shifted together, were no faster
// (77 x 2009 -> 5125: 15.6 us, 13.1 so).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ i8x16 load16(const int8_t* p) {
    const u32x4_any v = *(const __attribute__((address_space(1))) u32x4_any*)(p);
    return i8x16{(int)v.x, (int)v.y, (int)v.z, (int)v.w};
}

// Bytes k .. k + 15 of a row, zeros past K: one load that ends with the row at the latest, its
// bytes moved down.  (A byte at a time, each load waits for the one before: 77 x 2009 -> 5125 took
// 28 us.)  Only a row shorter than 16 bytes goes byte by byte.
__device__ __forceinline__ i8x16 load16_tail(const int8_t* row, int k, int K) {
    uint64_t lo = 0, hi = 0;
    if (K < 16) {
        for (int i = 0; k + i < K; ++i) {
            const uint64_t b = (uint8_t)row[k + i];
            if (i < 8) lo |= b << (8 * i);
            else hi |= b << (8 * (i - 8));
        }
    } else {
        const int at = min(k, K - 16), move = k - at;
        const i8x16 v = load16(row + at);
        lo = (uint32_t)v.x | ((uint64_t)(uint32_t)v.y << 32);
        hi = (uint32_t)v.z | ((uint64_t)(uint32_t)v.w << 32);
        if (move >= 8) {
            lo = hi;
            hi = 0;
        }
        const int bits = 8 * (move & 7);
        lo = (lo >> bits) | (bits ? hi << (64 - bits) : 0);
        hi >>= bits;
        if (move >= 16) lo = hi = 0;
    }
    return i8x16{(int)(uint32_t)lo, (int)(lo >> 32), (int)(uint32_t)hi, (int)(hi >> 32)};
}

// The affine of one output.  Rounded at the conversion, both products and the sum.
template <bool BIAS, bool SQRELU>
__device__ __forceinline__ float i8_affine(int acc, float as, float ws, float bias) {
    float v = __fmul_rn(__fmul_rn(static_cast<float>(acc), as), ws);
    if (BIAS) v = __fadd_rn(v, bias);
    if (SQRELU) {
        v = v < 0.0f ? 0.0f : v;  // a NaN stays
        v = __fmul_rn(v, v);
    }
    return v;
}

// Outputs n .. n + 3 of token m (of the segment) from their sums.
template <int YDT>
__device__ __forceinline__ void i8_store4(const I8Problem& pb, const I8Rows& rows, int n, int m,
                                          const i8x16& sum, void* __restrict__ y) {
    if (m >= rows.count || n >= pb.N) return;
    const int64_t orow = rows.begin + m;
    const float as = rows.act_scale[i8_source(rows, (int)orow)];
    float o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int at = min(n + c, pb.N - 1);
        const float ws = pb.w_scale[at];
        const float v = pb.bias ? i8_affine<true, false>(sum[c], as, ws, pb.bias[at])
                                : i8_affine<false, false>(sum[c], as, ws, 0.0f);
        const float h = v < 0.0f ? 0.0f : v;
        o[c] = pb.sqrelu ? __fmul_rn(h, h) : v;
    }
    const int64_t at = orow * pb.N + n;
    constexpr int kSize = YDT == NSOSX_F32 ? 4 : 2;
    char* dst = static_cast<char*>(y) + at * kSize;
    if (n + 4 <= pb.N && (reinterpret_cast<uintptr_t>(dst) & (4 * kSize - 1)) == 0) {
        if constexpr (YDT == NSOSX_F32)
            *reinterpret_cast<float4*>(dst) = make_float4(o[0], o[1], o[2], o[3]);
        else
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        return;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (n + c < pb.N) store_act<YDT>(y, at + c, o[c]);
}

// ===========================================================================
// Few tiles: a workgroup owns 16 NT outputs x 16 MT tokens, and its W waves each take a part of K
// for the whole tile, with v_mfma_i32_16x16x64_i8.  A wave has its own ring of D slots in LDS, a
// 64-deep block of the tile's 16 (NT + MT) rows each, so that nothing waits for another wave until
// the end, where the partial sums are added in LDS.
//
// The way through LDS is there for the loads: four neighbouring lanes fetch the 64 bytes of one
// row, which the vector cache serves at 60 bytes a clock, where lanes in the operand's order
// (neighbours on different rows) get 16.  A fragment's row r has its 16-byte chunk c in place
// c ^ (r / 4), so that the 16 lanes that read one chunk of 16 rows meet 64 different banks.  What
// bounds a tile is the wait for its loads: of 77 x 2009 -> 5125 the waves wait for 62 % of their time,
// LDS is busy for 18 % and the matrix units for 8 (on the compute units that have a tile).
// ===========================================================================
template <int NT, int MT, int W, int D>
constexpr int i8_split_smem() {
    const int ring = W * D * (NT + MT) * 1024, sums = W * NT * MT * 1024;
    return ring > sums ? ring : sums;
}

template <int YDT, int NT, int MT, int W, int D, bool ALIGNED>
__device__ __forceinline__ void i8_split_tile(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                              void* __restrict__ y, char* __restrict__ smem) {
    constexpr int F = NT + MT;  // fragments (16 rows x 64 bytes) of a block
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* ring = smem + wave * (D * F * 1024);
    // this lane's row and chunk of every fragment, as fetched
    const int fr = lane >> 2, fc = ((lane & 3) ^ (fr >> 2)) * 16;
    const int8_t* src[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        // rows past N or the segment re-read its last one; their outputs are not stored
        const int64_t row =
            f < NT ? min(n0 + 16 * f + fr, pb.N - 1)
                   : i8_source(rows, rows.begin + min(m0 + 16 * (f - NT) + fr, rows.count - 1));
        src[f] = (f < NT ? pb.w : rows.q) + row * pb.K;
    }
    // as read: row r, K quarter g
    const int r = lane & 15, g = lane >> 4;
    const int at = r * 64 + ((g ^ (r >> 2)) << 4);
    i8x16 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[n][t] = i8x16{0, 0, 0, 0};
    i8x16 fa[F];
    auto read = [&](int slot) {
#pragma unroll
        for (int f = 0; f < F; ++f) fa[f] = *reinterpret_cast<const i8x16*>(ring + (slot * F + f) * 1024 + at);
    };
    auto mul = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                acc[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[n], fa[NT + t], acc[n][t], 0, 0, 0);
    };
    const int full = pb.K / 64, blocks = (pb.K + 63) / 64;
    const int b0 = (int)((int64_t)blocks * wave / W), b1 = (int)((int64_t)blocks * (wave + 1) / W);
    const int e1 = min(b1, full);  // this wave's whole blocks: b0 .. e1 - 1
    if constexpr (ALIGNED) {
        auto issue = [&](int b, int slot) {
#pragma unroll
            for (int f = 0; f < F; ++f)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)(src[f] + b * 64 + fc),
                    (__attribute__((address_space(3))) void*)(ring + (slot * F + f) * 1024), 16, 0, 0);
        };
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (b0 + d < e1) issue(b0 + d, d);
        int slot = 0;
        for (int b = b0; b < e1; ++b) {
            if (b + D <= e1)  // D blocks are in flight: the oldest has landed
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * F) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            read(slot);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is read before it is filled
            if (b + D < e1) issue(b + D, slot);
            mul();
            slot = slot + 1 == D ? 0 : slot + 1;
        }
    } else {
        // through registers: the next block's loads lie under this one's products
        i8x16 reg[F];
#pragma unroll
        for (int f = 0; f < F; ++f)
            if (b0 < e1) reg[f] = load16(src[f] + b0 * 64 + fc);
        for (int b = b0; b < e1; ++b) {
#pragma unroll
            for (int f = 0; f < F; ++f) *reinterpret_cast<i8x16*>(ring + f * 1024 + lane * 16) = reg[f];
            if (b + 1 < e1)
#pragma unroll
                for (int f = 0; f < F; ++f) reg[f] = load16(src[f] + (b + 1) * 64 + fc);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            read(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            mul();
        }
    }
    if (b1 > full && b0 < b1) {  // the last block is not whole (every slot of the ring is free)
#pragma unroll
        for (int f = 0; f < F; ++f)
            *reinterpret_cast<i8x16*>(ring + f * 1024 + lane * 16) = load16_tail(src[f], full * 64 + fc, pb.K);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        read(0);
        mul();
    }
    // accumulator c of lane l: output n0 + 16 n + 4 (l / 16) + c, token m0 + 16 t + l % 16
    __syncthreads();  // every wave is done with its ring
    char* part = smem + wave * (NT * MT * 1024) + lane * 16;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<i8x16*>(part + (n * MT + t) * 1024) = acc[n][t];
    __syncthreads();
    for (int i = wave; i < NT * MT; i += W) {  // the waves share the 16 x 16 tiles out
        i8x16 sum = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < W; ++p)
            sum += *reinterpret_cast<const i8x16*>(smem + (p * NT * MT + i) * 1024 + lane * 16);
        i8_store4<YDT>(pb, rows, n0 + 16 * (i / MT) + 4 * g, m0 + 16 * (i % MT) + r, sum, y);
    }
}

// ===========================================================================
// Block tile: 64 NWN outputs x 32 TM NWM tokens, NWN x NWM waves of 64 x 32 TM = 2 x TM tiles
// of v_mfma_i32_32x32x32_i8, over 128-deep stages double-buffered in LDS.  A stage is fetched
// into registers while the one before it is multiplied.  16-byte chunk c of row r sits in slot
// c ^ ((r / 2) % 8), so that 16 neighbouring lanes of a ds_read_b128, 16 rows, lie in different
// banks.
// ===========================================================================
constexpr int kI8BK = 128;

// Two stages, and behind them the tile's scales and biases per output and scales per token, there
// from the start: fetched in the epilogue, they are two memory round trips of every tile.
template <int NWN, int NWM, int TM>
constexpr int i8_stages_smem() { return 2 * (64 * NWN + 32 * TM * NWM) * kI8BK; }
template <int NWN, int NWM, int TM>
constexpr int i8_tile_smem() {
    return i8_stages_smem<NWN, NWM, TM>() + (2 * 64 * NWN + 32 * TM * NWM) * 4;
}

template <int NWN, int NWM, int TM>
__device__ __forceinline__ void i8_stage_scales(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                                char* smem) {
    constexpr int kThreads = 64 * NWN * NWM, BN = 64 * NWN, BM = 32 * TM * NWM;
    float* s_scale = reinterpret_cast<float*>(smem + i8_stages_smem<NWN, NWM, TM>());
    for (int i = threadIdx.x; i < BN; i += kThreads) {
        const int n = min(n0 + i, pb.N - 1);
        s_scale[i] = pb.w_scale[n];
        if (pb.bias) s_scale[BN + i] = pb.bias[n];
    }
    for (int i = threadIdx.x; i < BM; i += kThreads)
        s_scale[2 * BN + i] = rows.act_scale[i8_source(rows, rows.begin + min(m0 + i, rows.count - 1))];
}

// Linear workgroup id -> tile.  Consecutive ids go round-robin to the 8 XCDs; each XCD takes a
// contiguous run of tiles, in bands of GM row tiles, rows fastest, so that the tiles in flight
// on an XCD share both operands in its L2 (128 x 128 tiles of 4096 x 4096 x 8192: 168 us with the
// outputs fastest, 150 in bands of 8).
template <int GM>
__device__ __forceinline__ void i8_tile_order(int L, int ntn, int ntm, int& nt, int& mt) {
    const int total = ntn * ntm, per = total / 8;
    const int t = L < per * 8 ? (L % 8) * per + L / 8 : L;
    const int band = t / (GM * ntn), first = band * GM, size = min(GM, ntm - first);
    const int in = t - first * ntn;
    mt = first + in % size;
    nt = in / size;
}

template <int YDT, int NWN, int NWM, int TM, bool BIAS, bool SQRELU>
__device__ __forceinline__ void i8_epilogue_as(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                            void* __restrict__ y, char* smem,
                                            const i32x16 (&acc)[2][TM]) {
    constexpr int kSize = YDT == NSOSX_F32 ? 4 : 2;
    constexpr int kRow = 64 * kSize, kSlice = 32 * kRow, kChunks = kRow / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wn = wave % NWN, wm = wave / NWN;
    const int g = lane >> 5, li = lane & 31;
    const float* s_scale = reinterpret_cast<const float*>(smem + i8_stages_smem<NWN, NWM, TM>());
    const float* s_bias = s_scale + 64 * NWN;
    const float* s_act = s_bias + 64 * NWN;
    float as[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) as[t] = s_act[32 * (wm * TM + t) + li];
    __syncthreads();  // every wave is done with the stages
    char* slice = smem + wave * kSlice;
    // 16-byte chunk c of row r sits in place c ^ swizzle(r): two rows of 128 bytes, or one of 256, are
    // all the banks
    auto swizzle = [](int row) { return YDT == NSOSX_F32 ? row & 15 : (row >> 1) & 7; };
    const int nw = n0 + 64 * wn;
    const bool whole = nw + 64 <= pb.N && pb.N % (16 / kSize) == 0 &&
                       (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    // the scales and biases of this lane's outputs, once for all TM tiles
    float4 sc[8], bs[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        sc[c] = *reinterpret_cast<const float4*>(s_scale + 64 * wn + 8 * c + 4 * g);
        bs[c] = BIAS ? *reinterpret_cast<const float4*>(s_bias + 64 * wn + 8 * c + 4 * g) : float4{};
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int mt = m0 + 32 * (wm * TM + t);
        if (mt >= rows.count) break;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const int at = 32 * nb + 8 * q4 + 4 * g;  // of the wave's 64 outputs
                const float4 s4 = sc[4 * nb + q4], b4 = bs[4 * nb + q4];
                const i32x16& a = acc[nb][t];
                const float o0 = i8_affine<BIAS, SQRELU>(a[4 * q4], as[t], s4.x, b4.x);
                const float o1 = i8_affine<BIAS, SQRELU>(a[4 * q4 + 1], as[t], s4.y, b4.y);
                const float o2 = i8_affine<BIAS, SQRELU>(a[4 * q4 + 2], as[t], s4.z, b4.z);
                const float o3 = i8_affine<BIAS, SQRELU>(a[4 * q4 + 3], as[t], s4.w, b4.w);
                char* dst = slice + li * kRow + ((at * kSize / 16 ^ swizzle(li)) << 4);
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
                    slice + row * kRow + ((c ^ swizzle(row)) << 4));
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
                                  ((((lane * kSize) / 16) ^ swizzle(row)) << 4) +
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

// (The branch on bias and activation is out here: inside, every output formed both and chose, and
// the epilogue's 9 operations an output, where 4 do, were 7 us of a 256 x 256 tile.)
template <int YDT, int NWN, int NWM, int TM>
__device__ __forceinline__ void i8_epilogue(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                            void* __restrict__ y, char* smem,
                                            const i32x16 (&acc)[2][TM]) {
    if (pb.sqrelu) {
        if (pb.bias) i8_epilogue_as<YDT, NWN, NWM, TM, true, true>(pb, rows, n0, m0, y, smem, acc);
        else i8_epilogue_as<YDT, NWN, NWM, TM, false, true>(pb, rows, n0, m0, y, smem, acc);
    } else {
        if (pb.bias) i8_epilogue_as<YDT, NWN, NWM, TM, true, false>(pb, rows, n0, m0, y, smem, acc);
        else i8_epilogue_as<YDT, NWN, NWM, TM, false, false>(pb, rows, n0, m0, y, smem, acc);
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
    i8_stage_scales<NWN, NWM, TM>(pb, rows, n0, m0, smem);
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

// The same tile with its stages brought straight into LDS (global_load_lds, 16 bytes a lane: the
// rows have to start on 16 bytes), and the last quarter of a stage multiplied after the barrier
// that frees its buffer, so that the barrier's wait and the first reads of the next stage lie
// under matrix instructions.  256 x 256 blocks of eight waves, 4096 x 4096 x 8192: 129 us,
// 2.1 POP/s (128 x 128 blocks 145, through registers 170 .. 178); matrix instructions alone reach
// 3.1 .. 3.5 POP/s on such data.  No unit bounds it by its rate: the matrix units are busy for 53 % of
// the clocks and LDS for 22 (4 clocks a ds_read_b128 of a wave); the two waves of a SIMD wait for 34 %
// of their time, at the stage's barrier and for its first reads.  64-deep stages in rings of three or
// four, and 256 x 128 blocks of four waves, two a compute unit, were no faster at any size (138 -> 142 ..
// 159 us).  At K 1024 the stores show, which all compute units make at once (8192 x 1024 x 4096: 43.5
// us, about 13 of them 67 MB of outputs).
template <int YDT, int NWN, int NWM, int TM>
__device__ __forceinline__ void i8_wide_tile(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                             void* __restrict__ y, char* smem) {
    constexpr int kWaves = NWN * NWM, BN = 64 * NWN, BM = 32 * TM * NWM;
    constexpr int kStage = (BN + BM) * kI8BK, kLoads = (BN + BM) / 8 / kWaves;
    static_assert(BN / 8 % kWaves == 0 && BM / 8 % kWaves == 0, "whole loads");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % NWN, wm = wave / NWN;
    const int g = lane >> 5, li = lane & 31;
    // load i of a wave fills rows 8 (i kWaves + wave) .. + 7 of the stage (weights, then tokens)
    const int8_t* src[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int row = (i * kWaves + wave) * 8 + (lane >> 3);
        const int c = (lane & 7) ^ ((row >> 1) & 7);
        // rows past N or the segment re-read its last one; their outputs are not stored
        src[i] = (i * kWaves * 8 < BN
                      ? pb.w + (int64_t)min(n0 + row, pb.N - 1) * pb.K
                      : rows.q + (int64_t)i8_source(rows, rows.begin + min(m0 + row - BN, rows.count - 1)) * pb.K) +
                 c * 16;
    }
    auto stage_at = [&](int kt, int i) { return smem + (kt & 1) * kStage + (i * kWaves + wave) * 1024; };
    auto issue = [&](int kt) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(src[i] + kt * kI8BK),
                (__attribute__((address_space(3))) void*)stage_at(kt, i), 16, 0, 0);
    };
    i32x16 acc[2][TM];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = i32x16{};
    const int sw = (li >> 1) & 7;
    const int wrow = (64 * wn + li) * kI8BK, xrow = (BN + 32 * TM * wm + li) * kI8BK;
    i8x16 fa[2][2], fb[2][TM];
    auto read = [&](int kt, int ks, int p) {
        const char* st = smem + (kt & 1) * kStage;
        const int slot = ((2 * ks + g) ^ sw) * 16;
#pragma unroll
        for (int n = 0; n < 2; ++n) fa[p][n] = *reinterpret_cast<const i8x16*>(st + wrow + n * 4096 + slot);
#pragma unroll
        for (int t = 0; t < TM; ++t) fb[p][t] = *reinterpret_cast<const i8x16*>(st + xrow + t * 4096 + slot);
    };
    auto mul = [&](int p) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int t = 0; t < TM; ++t)
                acc[n][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[p][n], fb[p][t], acc[n][t], 0, 0, 0);
    };
    // this wave's loads have landed and its reads are done; behind the barrier, everyone's
    auto meet = [&] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const int KT = pb.K / kI8BK;
    // a wave without outputs loads and meets with the others, and leaves the rest to them
    const bool busy = m0 + 32 * TM * wm < rows.count && n0 + 64 * wn < pb.N;
    if (KT > 0) issue(0);
    i8_stage_scales<NWN, NWM, TM>(pb, rows, n0, m0, smem);
    if (KT > 0) {
        meet();
        if (KT > 1) issue(1);
        if (busy) read(0, 0, 0);
    }
    for (int kt = 0; kt < KT; ++kt) {
        if (busy) {
            read(kt, 1, 1);
            mul(0);
            read(kt, 2, 0);
            mul(1);
            read(kt, 3, 1);
            mul(0);
        }
        meet();
        if (kt + 2 < KT) issue(kt + 2);
        if (busy) {
            if (kt + 1 < KT) read(kt + 1, 0, 0);
            mul(1);
        }
    }
    if (KT * kI8BK < pb.K) {
        // the last stage is not whole: through registers, zeros past K.  (Every wave has read every
        // stage into registers before the last barrier: both buffers are free.)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row = (i * kWaves + wave) * 8 + (lane >> 3);
            const int c = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
            *reinterpret_cast<i8x16*>(stage_at(KT, i) + lane * 16) =
                load16_tail(src[i] - c, KT * kI8BK + c, pb.K);
        }
        meet();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            read(KT, ks, 0);
            mul(0);
        }
    }
    i8_epilogue<YDT, NWN, NWM, TM>(pb, rows, n0, m0, y, smem, acc);
}

}  // namespace nsosx
