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

// W warps per row, VEC adjacent columns per access, CH accesses per thread: a thread holds columns (c * 32 W + t) * VEC + i
template <typename T, int W, int VEC, int CH>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 32)
k_norm_forward(const T* __restrict__ x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias, float eps,
               int64_t rows, int n, T* __restrict__ y, int64_t y_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int RB = W == 1 ? 8 : 1;  // rows per block
    __shared__ float s_sum[2][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * RB + (W == 1 ? warp : 0);
    if (row >= rows) return;
    const T* xr = x + row * x_stride;
    float v[CH][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * 32 * W + t) * VEC;
        if (col < n) {
            op_load<T, VEC>(xr + col, v[c]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[c][i] = 0.0f;
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += v[c][i];
    const float mean = norm_row_sum<W>(sum, s_sum[0], warp, lane) / (float)n;
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if ((c * 32 * W + t) * VEC < n) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = v[c][i] - mean;
                sq = fmaf(d, d, sq);
            }
        }
    }
    const float rstd = 1.0f / sqrtf(norm_row_sum<W>(sq, s_sum[1], warp, lane) / (float)n + eps);
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * y_stride;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * 32 * W + t) * VEC;
        if (col >= n) continue;
        float w[VEC], b[VEC], o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = weight ? weight[col + i] : 1.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) b[i] = bias ? bias[col + i] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = fmaf((v[c][i] - mean) * rstd, w[i], b[i]);
        op_store<T, VEC>(yr + col, o);
    }
}

// rows longer than NORM_REG_N: a block per row, three passes over it
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_forward_long(const T* __restrict__ x, int64_t x_stride, const float* __restrict__ weight, const float* __restrict__ bias, float eps, int n,
                    T* __restrict__ y, int64_t y_stride, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float s_sum[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T* xr = x + row * x_stride;
    float sum = 0.0f, sq = 0.0f;
    for (int c = threadIdx.x; c < n; c += 1024) sum += op_float(xr[c]);
    const float mean = norm_row_sum<32>(sum, s_sum[0], warp, lane) / (float)n;
    for (int c = threadIdx.x; c < n; c += 1024) {
        const float d = op_float(xr[c]) - mean;
        sq = fmaf(d, d, sq);
    }
    const float rstd = 1.0f / sqrtf(norm_row_sum<32>(sq, s_sum[1], warp, lane) / (float)n + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * y_stride;
    for (int c = threadIdx.x; c < n; c += 1024)
        yr[c] = op_round<T>(fmaf((op_float(xr[c]) - mean) * rstd, weight ? weight[c] : 1.0f, bias ? bias[c] : 0.0f));
}

// Backward: a block of W warps per row (W = 1: four rows side by side, a warp each) walks the rows block, block + grid, .. and keeps its
// columns' weight and bias gradients in registers; partial: [2][blocks][n].
template <typename T, int W, int VEC, int CH>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32)
k_norm_backward(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, const float* __restrict__ mean,
                const float* __restrict__ rstd, const float* __restrict__ weight, int64_t rows, int n, T* __restrict__ dx, int64_t dx_stride,
                float* __restrict__ partial) {
    constexpr int RB = W == 1 ? 4 : 1;
    __shared__ float s_sum[4][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane : threadIdx.x;
    float w[CH][VEC], aw[CH][VEC], ab[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (c * 32 * W + t) * VEC + i;
            w[c][i] = weight && col < n ? weight[col] : 1.0f;
            aw[c][i] = ab[c][i] = 0.0f;
        }
    const float inv_n = 1.0f / (float)n;
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * RB + (W == 1 ? warp : 0); row < rows; row += (int64_t)gridDim.x * RB, turn ^= 2) {
        const T *xr = x + row * x_stride, *gr = dy + row * dy_stride;
        float xv[CH][VEC], gv[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * 32 * W + t) * VEC;
            if (col < n) {
                op_load<T, VEC>(xr + col, xv[c]);
                op_load<T, VEC>(gr + col, gv[c]);
            }
        }
        const float mu = mean[row], r = rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if ((c * 32 * W + t) * VEC < n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (xv[c][i] - mu) * r, g = gv[c][i];
                    aw[c][i] = fmaf(g, xh, aw[c][i]);
                    ab[c][i] += g;
                    xv[c][i] = xh;
                    gv[c][i] = g * w[c][i];
                    s1 += gv[c][i];
                    s2 = fmaf(gv[c][i], xh, s2);
                }
            }
        }
        // two barriers' worth of buffers: a warp that is a row ahead writes the other pair
        s1 = op_group_sum<32>(s1);
        s2 = op_group_sum<32>(s2);
        if (W > 1) {
            if (lane == 0) {
                s_sum[turn][warp] = s1;
                s_sum[turn + 1][warp] = s2;
            }
            __syncthreads();
            s1 = s_sum[turn][0];
            s2 = s_sum[turn + 1][0];
#pragma unroll
            for (int k = 1; k < W; ++k) {
                s1 += s_sum[turn][k];
                s2 += s_sum[turn + 1][k];
            }
        }
        const float m1 = s1 * inv_n, m2 = s2 * inv_n;
        T* dr = dx + row * dx_stride;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * 32 * W + t) * VEC;
            if (col < n) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = r * (gv[c][i] - m1 - xv[c][i] * m2);
                op_store<T, VEC>(dr + col, o);
            }
        }
    }
    if (!partial) return;
    // W = 1: the four warps' sums are added in order, through the rows of the partials themselves (four per block)
    const int64_t prow = W == 1 ? (int64_t)blockIdx.x * RB + warp : blockIdx.x, prows = (int64_t)gridDim.x * RB;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int col = (c * 32 * W + t) * VEC + i;
            if (col < n) {
                partial[prow * n + col] = aw[c][i];
                partial[(prows + prow) * n + col] = ab[c][i];
            }
        }
}

// rows longer than NORM_REG_N_BACK: dx by a block per row, then the columns' sums by threads that walk down stripes of rows
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_backward_long(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, const float* __restrict__ mean,
                     const float* __restrict__ rstd, const float* __restrict__ weight, int n, T* __restrict__ dx, int64_t dx_stride) {
    __shared__ float s_sum[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *gr = dy + row * dy_stride;
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < n; c += 1024) {
        const float xh = (op_float(xr[c]) - mu) * r, t = op_float(gr[c]) * (weight ? weight[c] : 1.0f);
        s1 += t;
        s2 = fmaf(t, xh, s2);
    }
    const float m1 = norm_row_sum<32>(s1, s_sum[0], warp, lane) / (float)n, m2 = norm_row_sum<32>(s2, s_sum[1], warp, lane) / (float)n;
    T* dr = dx + row * dx_stride;
    for (int c = threadIdx.x; c < n; c += 1024) {
        const float xh = (op_float(xr[c]) - mu) * r, t = op_float(gr[c]) * (weight ? weight[c] : 1.0f);
        dr[c] = op_round<T>(r * (t - m1 - xh * m2));
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_columns_long(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x, int64_t x_stride, const float* __restrict__ mean,
                    const float* __restrict__ rstd, int64_t rows, int n, float* __restrict__ partial) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= n) return;
    float aw = 0.0f, ab = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = op_float(dy[row * dy_stride + col]);
        aw = fmaf(g, (op_float(x[row * x_stride + col]) - mean[row]) * rstd[row], aw);
        ab += g;
    }
    partial[(int64_t)blockIdx.y * n + col] = aw;
    partial[(int64_t)(gridDim.y + blockIdx.y) * n + col] = ab;
}

// dweight and dbias from the blocks' rows: 32 columns per block, warp w adds the rows w, w + 32, .., then the warps in order
__global__ void __launch_bounds__(1024) k_norm_columns_final(const float* __restrict__ partial, int prows, int n, float* __restrict__ dweight,
                                                              float* __restrict__ dbias) {
    __shared__ float s_sum[32][33];
    float* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    const float* p = partial + (int64_t)blockIdx.y * prows * n;
    float v = 0.0f;
    if (col < n)
#pragma unroll 4
        for (int r = warp; r < prows; r += 32) v += p[(int64_t)r * n + col];
    s_sum[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && col < n) {
        v = s_sum[0][lane];
#pragma unroll
        for (int w = 1; w < 32; ++w) v += s_sum[w][lane];
        out[col] = v;
    }
}

// Blocks of the backward pass.  More than a few rows per block, or the blocks' rows of gradients cost as much as the rows themselves;
// at most what runs at once.
int norm_backward_blocks(int64_t rows, int n) {
    if (n > NORM_REG_N_BACK) return (int)(rows < 64 ? (rows < 1 ? 1 : rows) : 64);
    const int64_t per = n <= 512 ? 4 : 1, most = (int64_t)sm_count() * (n <= 2048 ? 4 : 2);
    const int64_t want = (rows + 8 * per - 1) / (8 * per);
    return (int)(want < 1 ? 1 : want < most ? want : most);
}
int norm_partial_rows(int64_t rows, int n) { return norm_backward_blocks(rows, n) * (n <= 512 ? 4 : 1); }

template <typename T, int VEC, int W, int CH>
void norm_forward_go(cudaStream_t s, const void* x, int64_t xs, const float* w, const float* b, float eps, int64_t rows, int n, void* y, int64_t ys,
                     float* mean, float* rstd) {
    const int64_t blocks = W == 1 ? (rows + 7) / 8 : rows;
    k_norm_forward<T, W, VEC, CH><<<(unsigned)blocks, W == 1 ? 256 : W * 32, 0, s>>>((const T*)x, xs, w, b, eps, rows, n, (T*)y, ys, mean, rstd);
}
// A warp per row up to 2048 columns (no barrier in a row), eight warps above.
template <typename T, int VEC>
void norm_forward_pick(cudaStream_t s, const void* x, int64_t xs, const float* w, const float* b, float eps, int64_t rows, int n, void* y, int64_t ys,
                       float* mean, float* rstd) {
#define GO(W, K) \
    if (n <= (W) * (K) * 32) return norm_forward_go<T, VEC, W, ((K) + VEC - 1) / VEC>(s, x, xs, w, b, eps, rows, n, y, ys, mean, rstd)
    GO(1, 8); GO(1, 16); GO(1, 24); GO(1, 32); GO(1, 48); GO(1, 64);
    GO(8, 16); GO(8, 32); GO(16, 32);
#undef GO
    k_norm_forward_long<T><<<(unsigned)rows, 1024, 0, s>>>((const T*)x, xs, w, b, eps, n, (T*)y, ys, mean, rstd);
}

template <typename T, int VEC>
void norm_backward_pick(cudaStream_t s, const void* dy, int64_t dys, const void* x, int64_t xs, const float* mean, const float* rstd, const float* w,
                        int64_t rows, int n, void* dx, int64_t dxs, float* partial, int blocks) {
    // W warps x K columns per lane
#define GO(W, K)                                                                                                                              \
    if (n <= (W) * (K) * 32) {                                                                                                                \
        k_norm_backward<T, W, VEC, ((K) + VEC - 1) / VEC><<<(unsigned)blocks, W == 1 ? 128 : W * 32, 0, s>>>(                                  \
            (const T*)dy, dys, (const T*)x, xs, mean, rstd, w, rows, n, (T*)dx, dxs, partial);                                                \
        return;                                                                                                                               \
    }
    GO(1, 8) GO(1, 16) GO(4, 8) GO(4, 16) GO(8, 16) GO(16, 16)
#undef GO
    k_norm_backward_long<T><<<(unsigned)rows, 1024, 0, s>>>((const T*)dy, dys, (const T*)x, xs, mean, rstd, w, n, (T*)dx, dxs);
    if (partial)
        k_norm_columns_long<T><<<dim3((unsigned)ceil_div(n, 256), (unsigned)blocks), 256, 0, s>>>((const T*)dy, dys, (const T*)x, xs, mean, rstd, rows, n, partial);
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
    if (((uintptr_t)d_x | (uintptr_t)d_y) % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_x and d_y must be aligned to their elements");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = n % (16 / size) == 0 && norm_aligned(d_x, x_stride, size) && norm_aligned(d_y, y_stride, size);
#define ARGS s, d_x, x_stride, d_weight, d_bias, eps, rows, n, d_y, y_stride, d_mean, d_rstd
    if (type == TB_TYPE_F32) wide ? norm_forward_pick<float, 4>(ARGS) : norm_forward_pick<float, 1>(ARGS);
    else if (type == TB_TYPE_F16) wide ? norm_forward_pick<__half, 8>(ARGS) : norm_forward_pick<__half, 1>(ARGS);
    else wide ? norm_forward_pick<__nv_bfloat16, 8>(ARGS) : norm_forward_pick<__nv_bfloat16, 1>(ARGS);
#undef ARGS
    return op_launched(err, err_len);
}

extern "C" int64_t tb_layer_norm_backward_workspace(int64_t rows, int n) {
    if (rows < 0 || rows > NORM_MAX_ROWS || n < 1) return TB_ERR_INVALID_ARGUMENT;
    return (int64_t)norm_partial_rows(rows, n) * 2 * n * (int64_t)sizeof(float);
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
    if (((uintptr_t)d_dy | (uintptr_t)d_x | (uintptr_t)d_dx) % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must be aligned to their elements");
    const bool columns = d_dweight || d_dbias;
    if (columns && (!d_work || work_bytes < tb_layer_norm_backward_workspace(rows, n) || ((uintptr_t)d_work & 3)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)",
                         (long long)tb_layer_norm_backward_workspace(rows, n), (long long)work_bytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* partial = columns ? static_cast<float*>(d_work) : nullptr;
    const int blocks = norm_backward_blocks(rows, n);
    if (rows == 0) {
        if (d_dweight) cudaMemsetAsync(d_dweight, 0, (size_t)n * sizeof(float), s);
        if (d_dbias) cudaMemsetAsync(d_dbias, 0, (size_t)n * sizeof(float), s);
        return op_launched(err, err_len);
    }
    const bool wide = n % (16 / size) == 0 && norm_aligned(d_dy, dy_stride, size) && norm_aligned(d_x, x_stride, size) && norm_aligned(d_dx, dx_stride, size);
#define ARGS s, d_dy, dy_stride, d_x, x_stride, d_mean, d_rstd, d_weight, rows, n, d_dx, dx_stride, partial, blocks
    if (type == TB_TYPE_F32) wide ? norm_backward_pick<float, 4>(ARGS) : norm_backward_pick<float, 1>(ARGS);
    else if (type == TB_TYPE_F16) wide ? norm_backward_pick<__half, 8>(ARGS) : norm_backward_pick<__half, 1>(ARGS);
    else wide ? norm_backward_pick<__nv_bfloat16, 8>(ARGS) : norm_backward_pick<__nv_bfloat16, 1>(ARGS);
#undef ARGS
    if (columns) k_norm_columns_final<<<dim3((unsigned)ceil_div(n, 32), 2), 1024, 0, s>>>(partial, norm_partial_rows(rows, n), n, d_dweight, d_dbias);
    return op_launched(err, err_len);
}
