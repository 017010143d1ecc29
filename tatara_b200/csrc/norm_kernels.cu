// Layer norm of rows of features on the caller's device tensors, forward and backward.
//
//   forward    mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + eps),  y = (x - mean) * rstd * weight + bias
//   backward   xh = (x - mean) * rstd,  t = dy * weight,  dx = rstd * (t - mean(t) - xh * mean(t * xh)),
//              dweight = sum over rows of dy * xh,  dbias = sum over rows of dy
//
// Both are bound by memory: 8 (14) operations per element of a row that is read once (x; x and dy) and written once (y; dx).  A row
// stays in the registers of its threads between the passes over it, so the variance is a second sum of squared distances from the
// mean (no cancellation) at no traffic.  All sums are fp32: a thread's columns in ascending order, then halves of the lanes,
// then the warps in order.  The weight gradients are columns' sums: every block keeps those of its rows in registers over all
// of its rows, the blocks' rows are added in a fixed order by a second kernel, so that results repeat bit for bit.
//
// Measured (inputs not in L2): 65536 x 1536 fp32 forward 122 us (6.6 TB/s), backward 176 us (6.9 TB/s) and 9 us for the columns' sums; whole calls in a row,
// columns' sums included: 40000 x 2048 fp16 66 us (4.9 TB/s) and 107 us (4.6 TB/s): 16-bit rows are half the bytes for the same instructions, issue slots at 60 %.
// Rows that start anywhere, 35954 x 1175: fp32 63 us (5.4 TB/s) and 86 us (5.9 TB/s), bf16 55 and 83 (the gradient's first kernel 76).  256 x 256: one launch, 2 us.
#include "op_common.cuh"

namespace {

#define NORM_REG_N 16384     // longest row that the forward pass keeps in registers
#define NORM_REG_N_BACK 8192 // ... the backward pass, with two rows and three rows of columns' values

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

// Blocks of the kernels that walk down the rows which one SM holds: 24 warps of 80 registers.  Backward, fp16, 16384 x 768: 20.4 us; 30 warps of 64 (some
// spilled) 24.6, four rows at a time in 96 registers 26.0, the next rows fetched ahead in 175 registers 34.
constexpr int norm_per_sm(int warps, int all = 24) { return all / warps < 1 ? 1 : all / warps; }
// ... backward.  Four warps with a row each hold more of their own: 16 warps of 128 registers (200000 x 256 fp16: 71 us, with 24 warps 89)
constexpr int norm_per_sm_back(int warps) { return warps == 1 ? 4 : norm_per_sm(warps); }

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

// W warps per row, VEC adjacent columns per access, CH accesses per thread: a thread holds columns (c * LANES + t) * VEC + i.  With W = 1 a row has L lanes
// (8 or 16 for rows of up to 64 or 128 columns, or most lanes of a warp idle), which take R rows at once: those share the reads of weight and bias.
template <typename T, int W, int L, int VEC, int CH, int R>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32)
k_norm_forward(const T* x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias, float eps,
               int64_t rows, int n, T* y, int64_t y_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int LANES = W == 1 ? L : 32 * W, SUBS = W == 1 ? 32 / L : 1, RB = W == 1 ? 4 * SUBS * R : 1;  // rows per block
    __shared__ float s_sum[2][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane % L : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * RB + (W == 1 ? (warp * SUBS + lane / L) * R : 0);
    op_next_may_start();
    if (L == 32 && row >= rows) return;  // by whole warps; lanes that share a warp stay for its sums
    constexpr bool ALL = R == 1 && L == 32;
    OpRaw<T, VEC> v[R][CH];
    op_wait_for_previous();
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LANES + t) * VEC;
            if (col < n && (ALL || row + q < rows)) v[q][c].load(x + (row + q) * x_stride + col);
            else v[q][c].zero();
        }
    float mean[R], rstd[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        mean[q] = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) mean[q] += v[q][c].get(i);
    }
    norm_rows_sum<W, L, R>(mean, s_sum[0], warp, lane);
#pragma unroll
    for (int q = 0; q < R; ++q) {
        mean[q] /= (float)n;
        rstd[q] = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if ((c * LANES + t) * VEC < n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = v[q][c].get(i) - mean[q];
                    rstd[q] = fmaf(d, d, rstd[q]);
                }
            }
    }
    norm_rows_sum<W, L, R>(rstd, s_sum[1], warp, lane);
#pragma unroll
    for (int q = 0; q < R; ++q) {
        rstd[q] = 1.0f / sqrtf(rstd[q] / (float)n + eps);
        if (t == 0 && (ALL || row + q < rows)) {
            if (mean_out) mean_out[row + q] = mean[q];
            if (rstd_out) rstd_out[row + q] = rstd[q];
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LANES + t) * VEC;
        if (col >= n) continue;
        float w[VEC], b[VEC];
        norm_columns<VEC>(weight, col, 1.0f, w);
        norm_columns<VEC>(bias, col, 0.0f, b);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = fmaf((v[q][c].get(i) - mean[q]) * rstd[q], w[i], b[i]);
            if (ALL || row + q < rows) op_store<T, VEC>(y + (row + q) * y_stride + col, o);
        }
    }
}

// ---- rows that start anywhere: a thread's columns are single ones -----------------------------------------------------------
// How many of a thread's places are inside the row for every thread: W warps are the fewest that hold it with eight columns a thread, and sixteen with
// sixteen columns hold 4097 or more.
__host__ __device__ constexpr int norm_full(int warps, int vec, int places) { return vec * places == 16 ? places / 2 : places * (warps - 1) / warps; }

// Forward for rows over 256 columns that start anywhere: a block walks down the rows with its columns' weight and bias in registers, R rows at a time.
// 35954 x 1175: 64 us in fp32 (5.2 TB/s), 55 in bf16; with a warp per row, which reads weight and bias for every row and checks every column, 105 and 127.
// Two adjacent 16-bit columns per thread, one access where the row starts on a 4-byte boundary: 108 (the branch keeps the loads apart).
template <typename T, int W, int CH, int R>
__global__ void __launch_bounds__(W * 32, norm_per_sm(W, 32))
k_norm_forward_down(const T* x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias, float eps, int64_t rows, int n, T* y,
                    int64_t y_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int LANES = 32 * W, FULL = norm_full(W, 1, CH);
    __shared__ float s_sum[2][2][W][R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = threadIdx.x;
    float w[CH], b[CH];
    op_next_may_start();
    op_wait_for_previous();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = c * LANES + t;
        w[c] = weight && col < n ? weight[col] : 1.0f;
        b[c] = bias && col < n ? bias[col] : 0.0f;
    }
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * R; first < rows; first += (int64_t)gridDim.x * R, turn ^= 1) {
        OpRaw<T, 1> v[R][CH];
        float mean[R], rstd[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const T* xr = x + (first + q) * x_stride;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = c * LANES + t;
                v[q][c].zero();
                if (first + q < rows && (c < FULL || col < n)) v[q][c].load(xr + col);
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            mean[q] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c) mean[q] += v[q][c].get(0);
        }
        norm_block_sums<W, R>(mean, s_sum[turn][0], warp, lane);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            mean[q] /= (float)n;
            rstd[q] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float d = v[q][c].get(0) - mean[q];
                if (c < FULL || c * LANES + t < n) rstd[q] = fmaf(d, d, rstd[q]);
            }
        }
        norm_block_sums<W, R>(rstd, s_sum[turn][1], warp, lane);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            rstd[q] = 1.0f / sqrtf(rstd[q] / (float)n + eps);
            if (first + q >= rows) continue;
            if (t == 0) {
                if (mean_out) mean_out[first + q] = mean[q];
                if (rstd_out) rstd_out[first + q] = rstd[q];
            }
            T* yr = y + (first + q) * y_stride;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = c * LANES + t;
                if (c < FULL || col < n) yr[col] = op_round<T>(fmaf((v[q][c].get(0) - mean[q]) * rstd[q], w[c], b[c]));
            }
        }
    }
}

// rows longer than NORM_REG_N: a block per row, three passes over it.  C counts columns: int, or int64_t where the last step would go beyond 2^31 (64-bit columns
// cost the fp16 gradient of 2000 x 12288 10 %)
template <typename T, typename C>
__global__ void __launch_bounds__(1024)
k_norm_forward_long(const T* x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias, float eps, int n,
                    T* y, int64_t y_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float s_sum[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T* xr = x + row * x_stride;
    float sum = 0.0f, sq = 0.0f;
    op_next_may_start();
    op_wait_for_previous();
    for (C c = threadIdx.x; c < n; c += 1024) sum += op_float(xr[c]);
    const float mean = norm_row_sum<32>(sum, s_sum[0], warp, lane) / (float)n;
    for (C c = threadIdx.x; c < n; c += 1024) {
        const float d = op_float(xr[c]) - mean;
        sq = fmaf(d, d, sq);
    }
    const float rstd = 1.0f / sqrtf(norm_row_sum<32>(sq, s_sum[1], warp, lane) / (float)n + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * y_stride;
    for (C c = threadIdx.x; c < n; c += 1024)
        yr[c] = op_round<T>(fmaf((op_float(xr[c]) - mean) * rstd, weight ? weight[c] : 1.0f, bias ? bias[c] : 0.0f));
}

// Backward: a block of W warps per row (W = 1: rows side by side, L lanes each) takes R rows at a time, which shares one barrier, walks
// down the rows and keeps its columns' weight and bias gradients in registers; part_w, part_b: [blocks][n] (of a single block the gradients themselves),
// or both NULL.
// fp32, 65536 x 1536: 177 us, 6.8 TB/s.
template <typename T, int W, int L, int VEC, int CH, int R>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32, norm_per_sm_back(W))
k_norm_backward(const T* dy, int64_t dy_stride, const T* x, int64_t x_stride, const float* __restrict__ mean,
                const float* __restrict__ rstd, const float* __restrict__ weight, int64_t rows, int n, T* dx, int64_t dx_stride,
                float* __restrict__ part_w, float* __restrict__ part_b) {
    constexpr int FULL = norm_full(W, VEC, CH);
    // What is not there is read from the last row and columns and then set to zero, so that no branch keeps the loads apart: 16-bit rows of several warps
    // (16384 x 768 29.5 us, 27.6 so) and single columns of a warp (100000 x 201 120 us, 56 so).  fp32 and the others lose 0 to 20 %.
    constexpr bool CLAMP = sizeof(T) == 2 && (W > 1 ? VEC > 1 && W < 16 : VEC == 1 && L == 32);
    constexpr int LANES = W == 1 ? L : 32 * W, SUBS = W == 1 ? 32 / L : 1, RB = W == 1 ? 4 * SUBS : 1;
    __shared__ float s_sum[2][2 * R][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane % L : threadIdx.x;
    float w[CH][VEC], aw[CH][VEC], ab[CH][VEC];
    op_next_may_start();
    op_wait_for_previous();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LANES + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[c][i] = aw[c][i] = ab[c][i] = 0.0f;
        if (col < n) norm_columns<VEC>(weight, col, 1.0f, w[c]);
    }
    const float inv_n = 1.0f / (float)n;
    int turn = 0;
    // the lanes of a warp take the same number of turns
    for (int64_t turn0 = ((int64_t)blockIdx.x * RB + (W == 1 ? warp * SUBS : 0)) * R; turn0 < rows; turn0 += (int64_t)gridDim.x * RB * R, turn ^= 1) {
        const int64_t first = turn0 + (SUBS > 1 ? lane / L * R : 0);
        OpRaw<T, VEC> xv[R][CH], gv[R][CH];
        float mu[R], r[R], s1[R], s2[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const bool in = first + q < rows;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LANES + t) * VEC;
                const bool there = in && (c < FULL || col < n);
                if (CLAMP) {
                    const int64_t row = in ? first + q : rows - 1;
                    const int from = c < FULL ? col : min(col, n - VEC);
                    xv[q][c].load(x + row * x_stride + from);
                    gv[q][c].load(dy + row * dy_stride + from);
                }
                if (!CLAMP || !there) {
                    xv[q][c].zero();
                    gv[q][c].zero();
                }
                if (!CLAMP && there) {
                    xv[q][c].load(x + (first + q) * x_stride + col);
                    gv[q][c].load(dy + (first + q) * dy_stride + col);
                }
            }
            mu[q] = in ? mean[first + q] : 0.0f;
            r[q] = in ? rstd[first + q] : 0.0f;
        }
        // columns and rows that do not exist are zeros throughout: dy is, and so is whatever it is multiplied with
#pragma unroll
        for (int q = 0; q < R; ++q) {
            s1[q] = s2[q] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (xv[q][c].get(i) - mu[q]) * r[q], g = gv[q][c].get(i), gw = g * w[c][i];
                    aw[c][i] = fmaf(g, xh, aw[c][i]);
                    ab[c][i] += g;
                    s1[q] += gw;
                    s2[q] = fmaf(gw, xh, s2[q]);
                }
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
            for (int q = 0; q < R; ++q) {
                s1[q] += __shfl_xor_sync(0xffffffffu, s1[q], o);
                s2[q] += __shfl_xor_sync(0xffffffffu, s2[q], o);
            }
        if (W > 1) {
            // a warp that is a round ahead writes the other set
            if (lane == 0)
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    s_sum[turn][2 * q][warp] = s1[q];
                    s_sum[turn][2 * q + 1][warp] = s2[q];
                }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < R; ++q) {
                s1[q] = s_sum[turn][2 * q][0];
                s2[q] = s_sum[turn][2 * q + 1][0];
#pragma unroll
                for (int k = 1; k < W; ++k) {
                    s1[q] += s_sum[turn][2 * q][k];
                    s2[q] += s_sum[turn][2 * q + 1][k];
                }
            }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const float m1 = s1[q] * inv_n, m2 = s2[q] * inv_n;
            if (first + q < rows)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LANES + t) * VEC;
                    if (c < FULL || col < n) {
                        float o[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float xh = (xv[q][c].get(i) - mu[q]) * r[q];
                            o[i] = r[q] * (gv[q][c].get(i) * w[c][i] - m1 - xh * m2);
                        }
                        op_store<T, VEC>(dx + (first + q) * dx_stride + col, o);
                    }
                }
        }
    }
    if (!part_w) return;
    if (SUBS > 1)  // the rows of a warp, in halves
#pragma unroll
        for (int o = 16; o >= L; o >>= 1)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    aw[c][i] += __shfl_xor_sync(0xffffffffu, aw[c][i], o);
                    ab[c][i] += __shfl_xor_sync(0xffffffffu, ab[c][i], o);
                }
    if (W == 1) {  // the four warps' sums, in order
        __shared__ float s_acc[3][2][32 * CH * VEC];
        if (warp > 0)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    s_acc[warp - 1][0][(c * VEC + i) * 32 + lane] = aw[c][i];
                    s_acc[warp - 1][1][(c * VEC + i) * 32 + lane] = ab[c][i];
                }
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    aw[c][i] += s_acc[q][0][(c * VEC + i) * 32 + lane];
                    ab[c][i] += s_acc[q][1][(c * VEC + i) * 32 + lane];
                }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LANES + t) * VEC;
        if (col < n && (SUBS == 1 || lane < L)) {  // n is a multiple of VEC
            op_store<float, VEC>(part_w + (int64_t)blockIdx.x * n + col, aw[c]);
            op_store<float, VEC>(part_b + (int64_t)blockIdx.x * n + col, ab[c]);
        }
    }
}

// rows longer than NORM_REG_N_BACK: dx by a block per row, then the columns' sums by threads that walk down stripes of rows
template <typename T, typename C>
__global__ void __launch_bounds__(1024)
k_norm_backward_long(const T* dy, int64_t dy_stride, const T* x, int64_t x_stride, const float* __restrict__ mean,
                     const float* __restrict__ rstd, const float* __restrict__ weight, int n, T* dx, int64_t dx_stride) {
    __shared__ float s_sum[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *gr = dy + row * dy_stride;
    op_next_may_start();
    op_wait_for_previous();
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (C c = threadIdx.x; c < n; c += 1024) {
        const float xh = (op_float(xr[c]) - mu) * r, t = op_float(gr[c]) * (weight ? weight[c] : 1.0f);
        s1 += t;
        s2 = fmaf(t, xh, s2);
    }
    const float m1 = norm_row_sum<32>(s1, s_sum[0], warp, lane) / (float)n, m2 = norm_row_sum<32>(s2, s_sum[1], warp, lane) / (float)n;
    T* dr = dx + row * dx_stride;
    for (C c = threadIdx.x; c < n; c += 1024) {
        const float xh = (op_float(xr[c]) - mu) * r, t = op_float(gr[c]) * (weight ? weight[c] : 1.0f);
        dr[c] = op_round<T>(r * (t - m1 - xh * m2));
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_columns_long(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, const float* __restrict__ mean,
                    const float* __restrict__ rstd, int64_t rows, int n, float* __restrict__ part_w, float* __restrict__ part_b) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;  // may be beyond 2^31
    op_next_may_start();
    op_wait_for_previous();
    if (at >= (unsigned)n) return;
    const int col = (int)at;
    float aw = 0.0f, ab = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = op_float(dy[row * dy_stride + col]);
        aw = fmaf(g, (op_float(x[row * x_stride + col]) - mean[row]) * rstd[row], aw);
        ab += g;
    }
    part_w[(int64_t)blockIdx.y * n + col] = aw;
    part_b[(int64_t)blockIdx.y * n + col] = ab;
}

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
// Blocks: at most what runs at once; 16 rows or more for each, or the blocks' rows of gradients cost as much as the rows themselves, but
// one per SM as far as the rows go (256 rows of 256: 4 blocks took 12 us).
int norm_backward_blocks(int64_t rows, int n) {
    if (n > NORM_REG_N_BACK) return (int)(rows < 64 ? (rows < 1 ? 1 : rows) : 64);
    const int w = norm_warps(n);
    const int64_t turn = n <= 64 ? 32 : n <= 128 ? 16 : w == 1 ? 8 : 2, sms = sm_count(), most = sms * norm_per_sm_back(w);
    const int64_t turns = (rows + turn - 1) / turn, least = (16 + turn - 1) / turn, want = (turns + least - 1) / least;
    if (turns <= 2) return 1;  // no second launch then
    const int64_t few = turns < sms ? turns : sms, blocks = want < few ? few : want < most ? want : most;
    return (int)blocks;
}

// whether int counts a long row's columns, one step of 1024 beyond the last included
bool norm_counts(int n) { return n <= INT32_MAX - 1023; }

struct NormForward {
    cudaStream_t s;
    const void* x;
    int64_t xs;
    const float *w, *b;
    float eps;
    int64_t rows;
    int n;
    void* y;
    int64_t ys;
    float *mean, *rstd;
};
template <typename T, int VEC, int W, int L, int CH>
void norm_forward_go(const NormForward& a) {
    // registers of a row's share, and how many of its elements have to be on their way: two rows where that leaves the warps enough
    constexpr int R = W == 1 && CH * VEC * (int)sizeof(T) <= 64 ? 2 : 1;
    const int64_t per = W == 1 ? 128 / L * R : 1, blocks = (a.rows + per - 1) / per;
    op_launch_next(a.s, dim3((unsigned)blocks), dim3(W == 1 ? 128 : W * 32), 0, k_norm_forward<T, W, L, VEC, CH, R>, (const T*)a.x, a.xs, a.w, a.b, a.eps, a.rows, a.n, (T*)a.y, a.ys, a.mean, a.rstd);
}
template <typename T, int W, int CH, int R>
void norm_forward_down(const NormForward& a) {
    const int64_t want = (a.rows + R - 1) / R, most = (int64_t)sm_count() * norm_per_sm(W, 32);
    op_launch_next(a.s, dim3((unsigned)(want < most ? want : most)), dim3(W * 32), 0, k_norm_forward_down<T, W, CH, R>, (const T*)a.x, a.xs, a.w, a.b, a.eps, a.rows, a.n, (T*)a.y, a.ys, a.mean, a.rstd);
}
// Rows on 16-byte boundaries: 8, 16 or 32 lanes per row up to 64, 128 and 256 columns (200000 x 128 bf16 with 32 lanes 45 us, with 16 28.7), a warp up to
// 2048 columns of fp32 and 3072 of 16 bits (no barrier in a row; 30000 x 2560 bf16 72 us, with eight warps 94; 20000 x 4096 93 and 84), eight warps above.
// A block that walks down the rows with weight and bias in registers needs a barrier per sum: 40000 x 2048 fp16 88 us, a warp per row 72.
template <typename T, int VEC>
void norm_forward_pick(const NormForward& a) {
#define GO(W, L, K) \
    if (a.n <= (W) * (K) * (L)) return norm_forward_go<T, VEC, W, L, ((K) + VEC - 1) / VEC>(a)
    GO(1, 8, 8); GO(1, 16, 8); GO(1, 32, 8);
    if constexpr (VEC > 1) {
        if constexpr (VEC == 4) GO(1, 32, 12);
        GO(1, 32, 16); GO(1, 32, 24); GO(1, 32, 32); GO(1, 32, 40); GO(1, 32, 48); GO(1, 32, 56); GO(1, 32, 64);
        if constexpr (VEC == 8) { GO(1, 32, 80); GO(1, 32, 96); }
        GO(8, 32, 16); GO(8, 32, 32); GO(16, 32, 32);
    } else {
        if (a.n <= 4096) return norm_with_warps<2>(norm_warps(a.n), [&](auto w) { norm_forward_down<T, decltype(w)::value, 8, 2>(a); });
        if (a.n <= NORM_REG_N_BACK) return norm_forward_down<T, 16, 16, 1>(a);
    }
#undef GO
    op_launch_next(a.s, dim3((unsigned)a.rows), dim3(1024), 0, norm_counts(a.n) ? k_norm_forward_long<T, int> : k_norm_forward_long<T, int64_t>, (const T*)a.x, a.xs, a.w, a.b, a.eps, a.n, (T*)a.y, a.ys, a.mean, a.rstd);
}

struct NormBackward {
    cudaStream_t s;
    const void* dy;
    int64_t dys;
    const void* x;
    int64_t xs;
    const float *mean, *rstd, *w;
    int64_t rows;
    int n;
    void* dx;
    int64_t dxs;
    float *part_w, *part_b;
    int blocks;
};
template <typename T, int VEC, int W, int L, int CH, int R>
void norm_backward_go(const NormBackward& a) {
    op_launch_next(a.s, dim3((unsigned)a.blocks), dim3(W == 1 ? 128 : W * 32), 0, k_norm_backward<T, W, L, VEC, CH / VEC, R>, (const T*)a.dy, a.dys, (const T*)a.x, a.xs, a.mean, a.rstd, a.w, a.rows, a.n,
                                                                                                      (T*)a.dx, a.dxs, a.part_w, a.part_b);
}
template <typename T, int VEC>
void norm_backward_pick(const NormBackward& a) {
    if (a.n > NORM_REG_N_BACK) {
        // the columns first: dx may be dy's or x's memory
        if (a.part_w)
            op_launch_next(a.s, dim3((unsigned)ceil_div64(a.n, 256), (unsigned)a.blocks), dim3(256), 0, k_norm_columns_long<T>, (const T*)a.dy, a.dys, (const T*)a.x, a.xs, a.mean, a.rstd, a.rows, a.n, a.part_w,
                                                                                                             a.part_b);
        op_launch_next(a.s, dim3((unsigned)a.rows), dim3(1024), 0, norm_counts(a.n) ? k_norm_backward_long<T, int> : k_norm_backward_long<T, int64_t>, (const T*)a.dy, a.dys, (const T*)a.x, a.xs, a.mean, a.rstd, a.w, a.n, (T*)a.dx, a.dxs);
    } else if (a.n <= 64) {
        norm_backward_go<T, VEC, 1, 8, 8, 2>(a);
    } else if (a.n <= 128) {
        norm_backward_go<T, VEC, 1, 16, 8, 2>(a);
    } else if (a.n > 4096) {
        norm_backward_go<T, VEC, 16, 32, 16, 1>(a);
    } else {
        norm_with_warps<1>(norm_warps(a.n), [&](auto w) { norm_backward_go<T, VEC, decltype(w)::value, 32, 8, 2>(a); });
    }
}

bool norm_aligned(const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0; }

}  // namespace

#define NORM_MAX_ROWS 2147483647LL

extern "C" int tb_layer_norm_forward(const void* d_x, int64_t x_stride, const float* d_weight, const float* d_bias, float eps, int type,
                                     int64_t rows, int n, void* d_y, int64_t y_stride, float* d_mean, float* d_rstd, void* stream, char* err,
                                     size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int size = op_type_size(type);
    if (!size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (rows < 0 || rows > NORM_MAX_ROWS || n < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^31) and n positive");
    if (!(eps >= 0.0f)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "eps must not be negative");
    if (rows == 0) return TB_OK;
    if (!d_x || !d_y) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_x or d_y is NULL");
    if (rows > 1 && (x_stride < n || y_stride < n)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if (((uintptr_t)d_x | (uintptr_t)d_y) % size || ((uintptr_t)d_weight | (uintptr_t)d_bias | (uintptr_t)d_mean | (uintptr_t)d_rstd) & 3) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    if (!op_apart(d_x, 0, x_stride, d_y, 0, y_stride, 1, rows, n, size)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_y overlaps d_x in part");
    const OpRows xr = {d_x, x_stride * size, rows, (int64_t)n * size}, yr = {d_y, y_stride * size, rows, (int64_t)n * size};
    const OpRows wv = op_vector(d_weight, n), bv = op_vector(d_bias, n), mv = op_vector(d_mean, rows), rv = op_vector(d_rstd, rows);
    if (op_meets(yr, {wv, bv, mv, rv}) || op_meets(xr, {mv, rv}) || op_meets(wv, {mv, rv}) || op_meets(bv, {mv, rv}) || op_meets(mv, {rv}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = n % (16 / size) == 0 && norm_aligned(d_x, x_stride, size) && norm_aligned(d_y, y_stride, size) && (((uintptr_t)d_weight | (uintptr_t)d_bias) & 15) == 0;
    const NormForward a = {s, d_x, x_stride, d_weight, d_bias, eps, rows, n, d_y, y_stride, d_mean, d_rstd};
    if (type == TB_TYPE_F32) wide ? norm_forward_pick<float, 4>(a) : norm_forward_pick<float, 1>(a);
    else if (type == TB_TYPE_F16) wide ? norm_forward_pick<__half, 8>(a) : norm_forward_pick<__half, 1>(a);
    else wide ? norm_forward_pick<__nv_bfloat16, 8>(a) : norm_forward_pick<__nv_bfloat16, 1>(a);
    return op_launched(err, err_len);
}

extern "C" int64_t tb_layer_norm_backward_workspace(int64_t rows, int n) {
    if (rows < 0 || rows > NORM_MAX_ROWS || n < 1) return TB_ERR_INVALID_ARGUMENT;
    return (int64_t)norm_backward_blocks(rows, n) * 2 * n * (int64_t)sizeof(float);
}

extern "C" int tb_layer_norm_backward(const void* d_dy, int64_t dy_stride, const void* d_x, int64_t x_stride, const float* d_mean, const float* d_rstd,
                                      const float* d_weight, int type, int64_t rows, int n, void* d_dx, int64_t dx_stride, float* d_dweight,
                                      float* d_dbias, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int size = op_type_size(type);
    if (!size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (rows < 0 || rows > NORM_MAX_ROWS || n < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^31) and n positive");
    if (rows > 0 && (!d_dy || !d_x || !d_mean || !d_rstd || !d_dx)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (rows > 1 && (dy_stride < n || x_stride < n || dx_stride < n)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if (((uintptr_t)d_dy | (uintptr_t)d_x | (uintptr_t)d_dx) % size ||
        ((uintptr_t)d_weight | (uintptr_t)d_mean | (uintptr_t)d_rstd | (uintptr_t)d_dweight | (uintptr_t)d_dbias) & 3)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    if (rows > 0 && (!op_apart(d_dy, 0, dy_stride, d_dx, 0, dx_stride, 1, rows, n, size) || !op_apart(d_x, 0, x_stride, d_dx, 0, dx_stride, 1, rows, n, size)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dx overlaps d_dy or d_x in part");
    const bool columns = d_dweight || d_dbias;
    if (columns && (!d_work || work_bytes < tb_layer_norm_backward_workspace(rows, n) || ((uintptr_t)d_work & 31)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)",
                         (long long)tb_layer_norm_backward_workspace(rows, n), (long long)work_bytes);
    const OpRows wv = op_vector(d_weight, n), mv = op_vector(d_mean, rows), rv = op_vector(d_rstd, rows), dwv = op_vector(d_dweight, n), dbv = op_vector(d_dbias, n);
    const OpRows gr = {d_dy, dy_stride * size, rows, (int64_t)n * size}, xr = {d_x, x_stride * size, rows, (int64_t)n * size}, dr = {d_dx, dx_stride * size, rows, (int64_t)n * size};
    if (op_meets(dwv, {dbv}) || (rows > 0 && (op_meets(dr, {wv, mv, rv, dwv, dbv}) || op_meets(gr, {dwv, dbv}) || op_meets(xr, {dwv, dbv}) || op_meets(wv, {dwv, dbv}) ||
                                              op_meets(mv, {dwv, dbv}) || op_meets(rv, {dwv, dbv}))))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* partial = columns ? static_cast<float*>(d_work) : nullptr;
    const int blocks = norm_backward_blocks(rows, n);
    if (rows == 0) {
        if (d_dweight) op_note(cudaMemsetAsync(d_dweight, 0, (size_t)n * sizeof(float), s));
        if (d_dbias) op_note(cudaMemsetAsync(d_dbias, 0, (size_t)n * sizeof(float), s));
        return op_launched(err, err_len);
    }
    const bool wide = n % (16 / size) == 0 && norm_aligned(d_dy, dy_stride, size) && norm_aligned(d_x, x_stride, size) && norm_aligned(d_dx, dx_stride, size) && ((uintptr_t)d_weight & 15) == 0;
    // a single block writes the gradients themselves (its stores are as wide as 32 bytes)
    const bool direct = blocks == 1 && d_dweight && d_dbias && (((uintptr_t)d_dweight | (uintptr_t)d_dbias) & 31) == 0;
    const NormBackward a = {s, d_dy, dy_stride, d_x, x_stride, d_mean, d_rstd, d_weight, rows, n, d_dx, dx_stride, direct ? d_dweight : partial,
                            direct ? d_dbias : partial ? partial + (int64_t)blocks * n : nullptr, blocks};
    if (type == TB_TYPE_F32) wide ? norm_backward_pick<float, 4>(a) : norm_backward_pick<float, 1>(a);
    else if (type == TB_TYPE_F16) wide ? norm_backward_pick<__half, 8>(a) : norm_backward_pick<__half, 1>(a);
    else wide ? norm_backward_pick<__nv_bfloat16, 8>(a) : norm_backward_pick<__nv_bfloat16, 1>(a);
    if (columns && !direct) op_launch_next(s, dim3((unsigned)ceil_div64(n, 8), 2), dim3(1024), 0, k_norm_columns_final, partial, blocks, n, d_dweight, d_dbias);
    return op_launched(err, err_len);
}
