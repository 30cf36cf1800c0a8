// Products of int8 codes with int8 weights on gfx950, a scale per token and per output
// channel: y[m, n] = (sum_k q[m, k] w[n, k]) * act_scale[m] * w_scale[n] (+ bias[n]), for one
// weight matrix and for the row segments of a routed batch's experts.  The sums are exact in
// int32 (K <= 131071: 128 * 128 * K < 2^31), so every kernel here gives the same bits.
#include "int8_tiles.hpp"

#include <algorithm>

namespace nsosx {

// ---- one weight matrix ------------------------------------------------------

template <int YDT, int MT>
__global__ __launch_bounds__(kSkinnyThreads) void i8_skinny_kernel(I8Problem pb, I8Rows rows,
                                                                   void* __restrict__ y) {
    extern __shared__ __align__(16) char smem_i8[];
    const int ntn = (pb.N + 15) / 16;
    const int nt = blockIdx.x % ntn, mt = blockIdx.x / ntn;
    i8_skinny_tile<YDT, MT>(pb, rows, nt * 16, mt * 16 * MT, y,
                            reinterpret_cast<int32_t*>(smem_i8));
}

template <int YDT, int NWN, int NWM, int TM>
__global__ __launch_bounds__(64 * NWN * NWM) void i8_tile_kernel(I8Problem pb, I8Rows rows,
                                                                void* __restrict__ y) {
    extern __shared__ __align__(16) char smem_i8[];
    constexpr int BN = 64 * NWN, BM = 32 * TM * NWM;
    int nt, mt;
    i8_tile_order(blockIdx.x, (pb.N + BN - 1) / BN, (rows.count + BM - 1) / BM, nt, mt);
    i8_tile<YDT, NWN, NWM, TM>(pb, rows, nt * BN, mt * BM, y, smem_i8);
}

// ---- the experts' segments ----------------------------------------------------

template <int YDT, int MT>
__global__ __launch_bounds__(kSkinnyThreads) void i8_grouped_skinny_kernel(I8Group gp,
                                                                           void* __restrict__ y) {
    extern __shared__ __align__(16) char smem_i8[];
    const int ntn = (gp.N + 15) / 16;
    const int nt = blockIdx.x % ntn, e = blockIdx.x / ntn;
    I8Problem pb;
    I8Rows rows;
    if (!i8_segment(gp, e, pb, rows)) return;
    for (int m0 = 0; m0 < rows.count; m0 += 16 * MT) {
        i8_skinny_tile<YDT, MT>(pb, rows, nt * 16, m0, y, reinterpret_cast<int32_t*>(smem_i8));
        __syncthreads();  // the partial sums are read before the next tile's are written
    }
}

template <int YDT, int NWN, int NWM, int TM>
__global__ __launch_bounds__(64 * NWN * NWM) void i8_grouped_tile_kernel(I8Group gp,
                                                                        void* __restrict__ y) {
    extern __shared__ __align__(16) char smem_i8[];
    constexpr int BN = 64 * NWN, BM = 32 * TM * NWM;
    const int ntn = (gp.N + BN - 1) / BN;
    const int nt = blockIdx.x % ntn;
    int e, m0;
    if (!i8_find_segment<BM>(gp, blockIdx.x / ntn, e, m0)) return;
    I8Problem pb;
    I8Rows rows;
    if (!i8_segment(gp, e, pb, rows)) return;
    i8_tile<YDT, NWN, NWM, TM>(pb, rows, nt * BN, m0, y, smem_i8);
}

// ---- launches -------------------------------------------------------------------

template <int YDT, int MT>
static void launch_skinny_t(const I8Problem& pb, const I8Rows& rows, void* y, hipStream_t st) {
    const int64_t grid = (int64_t)((pb.N + 15) / 16) * ((rows.count + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((i8_skinny_kernel<YDT, MT>), dim3((unsigned)grid), dim3(kSkinnyThreads),
                       i8_skinny_smem(MT), st, pb, rows, y);
}

template <int YDT>
static void launch_int8(const I8Problem& pb, const I8Rows& rows, void* y, hipStream_t st) {
    if (rows.count <= 128) {
        if (rows.count <= 16) launch_skinny_t<YDT, 1>(pb, rows, y, st);
        else if (rows.count <= 32) launch_skinny_t<YDT, 2>(pb, rows, y, st);
        else launch_skinny_t<YDT, 4>(pb, rows, y, st);
        return;
    }
    const int64_t grid = (int64_t)((pb.N + 127) / 128) * ((rows.count + 127) / 128);
    hipLaunchKernelGGL((i8_tile_kernel<YDT, 2, 2, 2>), dim3((unsigned)grid), dim3(256),
                       (i8_tile_smem<2, 2, 2>()), st, pb, rows, y);
}

template <int YDT>
static void launch_grouped(const I8Group& gp, void* y, hipStream_t st) {
    if (gp.slots <= 64 * (int64_t)gp.experts) {
        const int64_t grid = (int64_t)((gp.N + 15) / 16) * gp.experts;
        hipLaunchKernelGGL((i8_grouped_skinny_kernel<YDT, 2>), dim3((unsigned)grid),
                           dim3(kSkinnyThreads), i8_skinny_smem(2), st, gp, y);
        return;
    }
    // every expert's last tile may be partial; a tile holds at least one row
    const int64_t mtiles = std::min<int64_t>(gp.slots, gp.slots / 128 + gp.experts);
    const int64_t grid = (int64_t)((gp.N + 127) / 128) * mtiles;
    hipLaunchKernelGGL((i8_grouped_tile_kernel<YDT, 2, 2, 2>), dim3((unsigned)grid), dim3(256),
                       (i8_tile_smem<2, 2, 2>()), st, gp, y);
}

}  // namespace nsosx

using namespace nsosx;

extern "C" int nsosx_int8_gemm(const int8_t* q, const float* act_scale, const int8_t* w,
                               const float* w_scale, const float* bias, int M, int K, int N,
                               void* y, int y_dtype, void* stream) {
    if (!q || !act_scale || !w || !w_scale || !y)
        return fail(NSOSX_ERR_INVALID, "int8_gemm: null pointer");
    if (M <= 0 || K <= 0 || N <= 0)
        return fail(NSOSX_ERR_INVALID, "int8_gemm: M, K and N must be positive");
    if (!valid_dtype(y_dtype)) return fail(NSOSX_ERR_INVALID, "int8_gemm: bad dtype");
    if (K > kI8MaxK) return fail(NSOSX_ERR_OVERFLOW, "int8_gemm: K past the int32 sums (131071)");
    if (((int64_t)N + 15) / 16 * (((int64_t)M + 15) / 16) > 0x7fffffffLL)
        return fail(NSOSX_ERR_OVERFLOW, "int8_gemm: M * N too large");
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
    if (((int64_t)N + 15) / 16 * ((int64_t)slots / 16 + experts) > 0x7fffffffLL)
        return fail(NSOSX_ERR_OVERFLOW, "grouped_int8_gemm: slots * N too large");
    const I8Group gp{w, w_scale, bias, q, act_scale, offsets, perm, q_rows, slots, experts, N, K,
                     squared_relu != 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (y_dtype == NSOSX_BF16) launch_grouped<NSOSX_BF16>(gp, y, st);
    else launch_grouped<NSOSX_F32>(gp, y, st);
    return check_launch("grouped_int8_gemm");
}
