// Shared by the norms of rows (norm_kernels.cu, rms_kernels.cu): sums over the threads of a row, columns' vectors, and the sums of columns over blocks.
#pragma once
#include "op_common.cuh"

#include <type_traits>

namespace {

// sum over the W warps of a row, the same bits in every thread; buf: a row's own [W] floats, not reused before the next barrier
template <int W>
__device__ __forceinline__ float norm_row_sum(float v, float* buf, int warp_in_row, int lane) {
    v = op_group_sum<32>(v);
    if (W == 1) return v;
    if (lane == 0) buf[warp_in_row] = v;
    __syncthreads();
    v = buf[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v += buf[w];
    return v;
}

// the same of R rows of L lanes (R = 1 with several warps per row), in place
template <int W, int L, int R>
__device__ __forceinline__ void norm_rows_sum(float (&v)[R], float* buf, int warp_in_row, int lane) {
    if (W > 1) {
        v[0] = norm_row_sum<W>(v[0], buf, warp_in_row, lane);
        return;
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int q = 0; q < R; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
}

// the sums of R rows over the W warps of a block, in place; buf is not written again before the next barrier but one
template <int W, int R>
__device__ __forceinline__ void norm_block_sums(float (&v)[R], float (*buf)[R], int warp, int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int q = 0; q < R; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
    if (lane == 0)
#pragma unroll
        for (int q = 0; q < R; ++q) buf[warp][q] = v[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < R; ++q) v[q] = buf[0][q];
#pragma unroll
    for (int k = 1; k < W; ++k)
#pragma unroll
        for (int q = 0; q < R; ++q) v[q] += buf[k][q];
}

// VEC columns of a weight or bias, in 16-byte accesses (one element at a time they cost four to eight times the L1 wavefronts of the row
// itself: 24 -> 8 us for 10000 rows of 1000 fp16)
template <int VEC>
__device__ __forceinline__ void norm_columns(const float* __restrict__ p, int col, float none, float (&to)[VEC]) {
    constexpr int STEP = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int i = 0; i < VEC; i += STEP) {
        float t[STEP];
#pragma unroll
        for (int k = 0; k < STEP; ++k) t[k] = none;
        if (p) op_load<float, STEP>(p + col + i, t);
#pragma unroll
        for (int k = 0; k < STEP; ++k) to[i + k] = t[k];
    }
}

// How many of a thread's places are inside the row for every thread: W warps are the fewest that hold it with eight columns a thread, and sixteen with
// sixteen columns hold 4097 or more.
__host__ __device__ constexpr int norm_full(int warps, int vec, int places) { return vec * places == 16 ? places / 2 : places * (warps - 1) / warps; }

// dweight and dbias from the blocks' rows: eight columns (a 32-byte sector) per block; thread group r of 128 adds the rows r, r + 128, .., the four
// groups of a warp are added in halves, then the warps in halves.
__global__ void __launch_bounds__(1024) k_norm_columns_final(const float* __restrict__ partial, int prows, int n, float* __restrict__ dweight,
                                                              float* __restrict__ dbias) {
    __shared__ float s_sum[32][9];
    float* out = blockIdx.y ? dbias : dweight;
    op_next_may_start();
    if (!out) return;  // of the same block all
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = threadIdx.x & 7;
    const unsigned col = blockIdx.x * 8 + c;
    const float* p = partial + (int64_t)blockIdx.y * prows * n;
    float v = 0.0f;
    op_wait_for_previous();
    if (col < (unsigned)n)
        for (int r0 = threadIdx.x >> 3; r0 < prows; r0 += 128 * 8) {
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = r0 + 128 * i < prows ? p[(int64_t)(r0 + 128 * i) * n + col] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) v += t[i];
        }
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    if (lane < 8) s_sum[warp][c] = v;
    __syncthreads();
    if (warp >= 8) return;
    v = op_group_sum<32>(s_sum[lane][warp]);
    if (lane == 0 && blockIdx.x * 8 + warp < (unsigned)n) out[blockIdx.x * 8 + warp] = v;
}

// Warps per row of the kernels that walk down the rows: the fewest that hold it with eight columns a thread (up to 4096 columns, two rows at a time),
// sixteen with sixteen columns (one row) up to 8192.
int norm_warps(int n) { return n <= 4096 ? (n + 255) / 256 : 16; }
template <int FROM, typename F>
void norm_with_warps(int w, F&& f) {  // f(std::integral_constant<int, W>)
    if constexpr (FROM <= 16) {
        if (w == FROM) f(std::integral_constant<int, FROM>());
        else norm_with_warps<FROM + 1>(w, f);
    }
}
bool norm_aligned(const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0; }


}  // namespace
