// Products of int8 codes with int8 weights on gfx950, a scale per token and per output
// channel: y[m, n] = (sum_k q[m, k] w[n, k]) * act_scale[m] * w_scale[n] (+ bias[n]), for one
// weight matrix and for the row segments of a routed batch's experts.  The sums are exact in
// int32 (K <= 131071: 128 * 128 * K < 2^31), so every kernel here gives the same bits.
#include "int8_tiles.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nsosx {

// The tiles of a kernel: kN outputs x kM tokens a workgroup.
template <int NT, int MT, int W, int D, bool ALIGNED>
struct Split {
    static constexpr int kN = 16 * NT, kM = 16 * MT, kThreads = 64 * W;
    static constexpr int kBand = 8, kWavesPerSimd = 1;
    static constexpr bool kRuns = false;
    static constexpr int kSmem = i8_split_smem<NT, MT, W, D>();
    template <int YDT>
    static __device__ __forceinline__ void run(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                               void* y, char* smem) {
        i8_split_tile<YDT, NT, MT, W, D, ALIGNED>(pb, rows, n0, m0, y, smem);
    }
};

template <int NWN, int NWM, int TM>
struct Staged {  // any alignment
    static constexpr int kN = 64 * NWN, kM = 32 * TM * NWM, kThreads = 64 * NWN * NWM;
    static constexpr int kBand = 8, kWavesPerSimd = 1;
    static constexpr bool kRuns = true;
    static constexpr int kSmem = i8_tile_smem<NWN, NWM, TM>();
    template <int YDT>
    static __device__ __forceinline__ void run(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                               void* y, char* smem) {
        i8_tile<YDT, NWN, NWM, TM>(pb, rows, n0, m0, y, smem);
    }
};

template <int NWN, int NWM, int TM, int BAND, int WPS>
struct Wide {  // 16-byte aligned rows
    static constexpr int kN = 64 * NWN, kM = 32 * TM * NWM, kThreads = 64 * NWN * NWM;
    static constexpr int kBand = BAND, kWavesPerSimd = WPS;
    static constexpr bool kRuns = true;
    static constexpr int kSmem = i8_tile_smem<NWN, NWM, TM>();
    template <int YDT>
    static __device__ __forceinline__ void run(const I8Problem& pb, const I8Rows& rows, int n0, int m0,
                                               void* y, char* smem) {
        i8_wide_tile<YDT, NWN, NWM, TM>(pb, rows, n0, m0, y, smem);
    }
};

template <bool A> using Split16x16 = Split<1, 1, 8, 4, A>;
template <bool A> using Split16x64 = Split<1, 4, 8, 3, A>;
template <bool A> using Split32x64 = Split<2, 4, 4, 3, A>;
template <bool A> using Split64x64 = Split<4, 4, 4, 4, A>;
using Block128 = Wide<2, 2, 2, 8, 2>;
using Block256 = Wide<4, 2, 4, 4, 1>;
using Any128 = Staged<2, 2, 2>;

// ---- one weight matrix ------------------------------------------------------

template <class T, int YDT>
__global__ __launch_bounds__(T::kThreads, T::kWavesPerSimd) void i8_gemm_kernel(I8Problem pb, I8Rows rows,
                                                                              void* __restrict__ y) {
    extern __shared__ __align__(1024) char smem_i8[];
    int nt, mt;
    i8_tile_order<T::kBand>(blockIdx.x, (pb.N + T::kN - 1) / T::kN, (rows.count + T::kM - 1) / T::kM, nt, mt);
    T::template run<YDT>(pb, rows, nt * T::kN, mt * T::kM, y, smem_i8);
}

// ---- the experts' segments ----------------------------------------------------

// One row tile of one segment a workgroup.  Outputs are fastest, so that where their tiles divide
// by the 8 XCDs, each XCD reads an eighth of every expert's weights.  Where they do not, and an
// expert has more than one row tile to share its weights, the large tiles are dealt to the XCDs in
// contiguous runs, as those of one matrix, so that they are read by one or two (128 x 128 tiles,
// 8192 rows to 8 of 128 experts of 2048 -> 768: 169 us, and 200 with outputs fastest; to 2 of 8
// experts of 1024 -> 4096, whose tiles do divide: 112 and 105).  The launch holds as many
// workgroups as there can be tiles; those past the real ones end here.
template <class T, int YDT>
__global__ __launch_bounds__(T::kThreads, T::kWavesPerSimd) void i8_grouped_kernel(I8Group gp,
                                                                                 void* __restrict__ y) {
    extern __shared__ __align__(1024) char smem_i8[];
    const int ntn = (gp.N + T::kN - 1) / T::kN;
    int nt = blockIdx.x % ntn, mt = blockIdx.x / ntn;
    if (T::kRuns && ntn % 8 != 0 && gp.slots > (int64_t)T::kM * gp.experts) {
        const int total = i8_all_tiles<T::kM>(gp);
        if (mt >= total) return;
        i8_tile_order<T::kBand>(blockIdx.x, ntn, total, nt, mt);
    }
    int e, m0;
    if (!i8_find_segment<T::kM>(gp, mt, e, m0)) return;
    I8Problem pb;
    I8Rows rows;
    if (!i8_segment(gp, e, pb, rows)) return;
    T::template run<YDT>(pb, rows, nt * T::kN, m0, y, smem_i8);
}

// ---- launches -------------------------------------------------------------------

template <class T, int YDT>
static void launch_gemm_t(const I8Problem& pb, const I8Rows& rows, void* y, hipStream_t st) {
    const int64_t grid = (int64_t)((pb.N - 1) / T::kN + 1) * ((rows.count - 1) / T::kM + 1);
    hipLaunchKernelGGL((i8_gemm_kernel<T, YDT>), dim3((unsigned)grid), dim3(T::kThreads), T::kSmem, st,
                       pb, rows, y);
}

template <class T, int YDT>
static void launch_grouped_t(const I8Group& gp, void* y, hipStream_t st) {
    // every expert's last tile may be partial, and a tile holds at least one row
    const int64_t mtiles = std::min<int64_t>(gp.slots, gp.slots / T::kM + gp.experts);
    const int64_t grid = (int64_t)((gp.N - 1) / T::kN + 1) * mtiles;
    hipLaunchKernelGGL((i8_grouped_kernel<T, YDT>), dim3((unsigned)grid), dim3(T::kThreads), T::kSmem,
                       st, gp, y);
}

// Which tile takes a shape: the estimated time of each in us, fitted to sweeps of K 64 .. 8192,
// N 16 .. 8192 and 1 .. 16384 rows with the weights from HBM (330 shapes, of one matrix: within 10 % of
// the measured times on average, and the choice within 1 % of the best one's time on average, 27 % at
// most; experts whose rows are very uneven were not among them): a fixed part
// and one per round of 256 tiles, linear in K but no less than the tile's outputs and its
// start take.  A round is a whole one where a compute unit holds one workgroup.  Measured, us (16 x
// 16 / 16 x 64 / 32 x 64 / 64 x 64 / 128 x 128 / 256 x 256):
//   K 4096, N 4096:    1 row   5.1 /  5.9 /  6.8 / 10.0 / 21   / 47
//                     64 rows 10.7 / 11.1 /  9.6 / 12.5 / 23   / 49
//                    200 rows    - / 29   / 16.8 / 14.1 / 23   / 51
//                   1024 rows    - /  -   / 52   / 48   / 26   / 52
//                   4096 rows    - /  -   /  -   /  -   / 72   / 66
//   K 64, N 4096:     16 rows  3.1 /  3.4 /  3.7 /  5.0 /  5.1 /  6.0
//                    449 rows 26   / 18   /  7.4 /  9.4 /  6.4 /  8.7
//                   8000 rows    - /  -   /  -   /  -   / 23   / 20
// Rows that do not start on 16 bytes go through registers on the way to LDS, which costs every
// tile about a quarter, and have no 256 x 256 one (2048 x 2009 -> 5125 on 128 x 128: 55 us).
constexpr int64_t kI8MaxTiles = 1 << 24;  // of 128 x 128: 256 threads each, less than 2^32
constexpr int kI8MaxSide = 1 << 30;       // a tile's first row or output, and what it adds, in int

// (experts 0: one matrix)
static bool too_large(int rows, int N, int experts) {
    const int64_t mtiles = experts ? (int64_t)rows / 128 + experts : ((int64_t)rows + 127) / 128;
    return rows > kI8MaxSide || N > kI8MaxSide || ((int64_t)N + 127) / 128 * mtiles >= kI8MaxTiles;
}

enum class I8Tile { k16x16, k16x64, k32x64, k64x64, k128x128, k256x256 };

template <class Tiles>
static I8Tile choose_tile(int K, bool aligned, Tiles tiles) {
    const double k = K / 1024.0;
    auto part = [](double t) { return std::max(1.0, t / 256); };
    auto whole = [](double t) { return std::max(1.0, std::ceil(t / 256)); };
    const double cost[] = {
        2.2 - 0.15 * k + part(tiles(16, 16)) * std::max(0.9, 0.7 + 0.45 * k),
        1.6 - k + whole(tiles(16, 64)) * std::max(2.3, 1.64 + 1.75 * k),
        2.6 - 0.4 * k + whole(tiles(32, 64)) * std::max(1.4, 0.6 + 1.66 * k),
        1.0 - 0.5 * k + whole(tiles(64, 64)) * std::max(4.0, 3.25 + 2.43 * k),
        2.7 + 0.8 * k + part(tiles(128, 128)) * std::max(2.6, 1.2 + 4.2 * k),
        whole(tiles(256, 256)) * std::max(10.0, 6.8 + 14.7 * k),
    };
    // a launch holds less than 2^32 threads (tiles of 16 rows: 512 each): the larger ones always do
    const bool fits[] = {tiles(16, 16) < 4e6, tiles(16, 64) < 4e6, tiles(32, 64) < 8e6,
                         tiles(64, 64) < 8e6, true, aligned};
    int best = 4;
    for (int i = 0; i < 6; ++i)
        if (fits[i] && cost[i] < cost[best]) best = i;
    return static_cast<I8Tile>(best);
}

// The tile of M rows and one weight matrix.
static I8Tile matrix_tile(int M, int K, int N, bool aligned) {
    return choose_tile(K, aligned, [&](int n, int m) {
        return (double)((N - 1) / n + 1) * ((M - 1) / m + 1);
    });
}

// The tile of the experts' slots, whose counts are on the device: each expert's last tile is taken
// as three quarters of a tile more than its share.
static I8Tile experts_tile(int slots, int K, int N, int experts, bool aligned) {
    return choose_tile(K, aligned, [&](int n, int m) {
        return (double)((N - 1) / n + 1) *
               std::min<double>(slots, std::ceil((double)slots / m + 0.75 * experts));
    });
}

template <int YDT, bool A>
static void launch_int8_t(const I8Problem& pb, const I8Rows& rows, void* y, hipStream_t st) {
    switch (matrix_tile(rows.count, pb.K, pb.N, A)) {
        case I8Tile::k16x16: return launch_gemm_t<Split16x16<A>, YDT>(pb, rows, y, st);
        case I8Tile::k16x64: return launch_gemm_t<Split16x64<A>, YDT>(pb, rows, y, st);
        case I8Tile::k32x64: return launch_gemm_t<Split32x64<A>, YDT>(pb, rows, y, st);
        case I8Tile::k64x64: return launch_gemm_t<Split64x64<A>, YDT>(pb, rows, y, st);
        case I8Tile::k128x128:
            return launch_gemm_t<std::conditional_t<A, Block128, Any128>, YDT>(pb, rows, y, st);
        case I8Tile::k256x256:
            if constexpr (A) launch_gemm_t<Block256, YDT>(pb, rows, y, st);
    }
}

template <int YDT, bool A>
static void launch_grouped_a(const I8Group& gp, void* y, hipStream_t st) {
    switch (experts_tile(gp.slots, gp.K, gp.N, gp.experts, A)) {
        case I8Tile::k16x16: return launch_grouped_t<Split16x16<A>, YDT>(gp, y, st);
        case I8Tile::k16x64: return launch_grouped_t<Split16x64<A>, YDT>(gp, y, st);
        case I8Tile::k32x64: return launch_grouped_t<Split32x64<A>, YDT>(gp, y, st);
        case I8Tile::k64x64: return launch_grouped_t<Split64x64<A>, YDT>(gp, y, st);
        case I8Tile::k128x128:
            return launch_grouped_t<std::conditional_t<A, Block128, Any128>, YDT>(gp, y, st);
        case I8Tile::k256x256:
            if constexpr (A) launch_grouped_t<Block256, YDT>(gp, y, st);
    }
}

// rows that all start on 16 bytes
static bool aligned_rows(int K, const void* a, const void* b) {
    return K % 16 == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

template <int YDT>
static void launch_int8(const I8Problem& pb, const I8Rows& rows, void* y, hipStream_t st) {
    if (aligned_rows(pb.K, pb.w, rows.q)) launch_int8_t<YDT, true>(pb, rows, y, st);
    else launch_int8_t<YDT, false>(pb, rows, y, st);
}

template <int YDT>
static void launch_grouped(const I8Group& gp, void* y, hipStream_t st) {
    if (aligned_rows(gp.K, gp.w, gp.q)) launch_grouped_a<YDT, true>(gp, y, st);
    else launch_grouped_a<YDT, false>(gp, y, st);
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int nsosx_int8_gemm_tile(int rows, int K, int N, int experts, int aligned) {
    if (rows <= 0 || K <= 0 || K > kI8MaxK || N <= 0 || experts < 0 || experts > kI8MaxExperts ||
        too_large(rows, N, experts))
        return -1;
    const bool a = aligned && K % 16 == 0;
    return static_cast<int>(experts ? experts_tile(rows, K, N, experts, a) : matrix_tile(rows, K, N, a));
}

extern "C" int nsosx_int8_gemm(const int8_t* q, const float* act_scale, const int8_t* w,
                               const float* w_scale, const float* bias, int M, int K, int N,
                               void* y, int y_dtype, void* stream) {
    if (!q || !act_scale || !w || !w_scale || !y)
        return fail(NSOSX_ERR_INVALID, "int8_gemm: null pointer");
    if (M <= 0 || K <= 0 || N <= 0)
        return fail(NSOSX_ERR_INVALID, "int8_gemm: M, K and N must be positive");
    if (!valid_dtype(y_dtype)) return fail(NSOSX_ERR_INVALID, "int8_gemm: bad dtype");
    if (K > kI8MaxK) return fail(NSOSX_ERR_OVERFLOW, "int8_gemm: K past the int32 sums (131071)");
    if (too_large(M, N, 0))
        return fail(NSOSX_ERR_OVERFLOW, "int8_gemm: M, N or M * N too large");
    const int64_t yb = (int64_t)M * N * (y_dtype == NSOSX_F32 ? 4 : 2);
    if (overlaps(y, yb, q, (int64_t)M * K) || overlaps(y, yb, w, (int64_t)N * K))
        return fail(NSOSX_ERR_INVALID, "int8_gemm: y overlaps an input");
    const I8Problem pb{w, w_scale, bias, N, K, 0};
    const I8Rows rows{q, act_scale, nullptr, 0, M, M};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (y_dtype == NSOSX_BF16) launch_int8<NSOSX_BF16>(pb, rows, y, st);
    else launch_int8<NSOSX_F32>(pb, rows, y, st);
    return check_launch("int8_gemm");
}

extern "C" int nsosx_grouped_int8_gemm(const int8_t* q, const float* act_scale, int q_rows,
                                       const int8_t* w, const float* w_scale, const float* bias,
                                       const int32_t* offsets, const int32_t* perm, int slots,
                                       int experts, int K, int N, int squared_relu, void* y,
                                       int y_dtype, void* stream) {
    if (!q || !act_scale || !w || !w_scale || !offsets || !y)
        return fail(NSOSX_ERR_INVALID, "grouped_int8_gemm: null pointer");
    if (q_rows <= 0 || slots <= 0 || K <= 0 || N <= 0 || experts <= 0 || experts > kI8MaxExperts)
        return fail(NSOSX_ERR_INVALID,
                    "grouped_int8_gemm: sizes must be positive and experts <= 1024");
    if (!perm && q_rows < slots)
        return fail(NSOSX_ERR_INVALID, "grouped_int8_gemm: without perm q must hold every slot");
    if (!valid_dtype(y_dtype)) return fail(NSOSX_ERR_INVALID, "grouped_int8_gemm: bad dtype");
    if (K > kI8MaxK)
        return fail(NSOSX_ERR_OVERFLOW, "grouped_int8_gemm: K past the int32 sums (131071)");
    if (too_large(slots, N, experts))
        return fail(NSOSX_ERR_OVERFLOW, "grouped_int8_gemm: slots, N or slots * N too large");
    const int64_t yb = (int64_t)slots * N * (y_dtype == NSOSX_F32 ? 4 : 2);
    if (overlaps(y, yb, q, (int64_t)q_rows * K) || overlaps(y, yb, w, (int64_t)experts * N * K))
        return fail(NSOSX_ERR_INVALID, "grouped_int8_gemm: y overlaps an input");
    const I8Group gp{w, w_scale, bias, q, act_scale, offsets, perm, q_rows, slots, experts, N, K,
                     squared_relu != 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (y_dtype == NSOSX_BF16) launch_grouped<NSOSX_BF16>(gp, y, st);
    else launch_grouped<NSOSX_F32>(gp, y, st);
    return check_launch("grouped_int8_gemm");
}
