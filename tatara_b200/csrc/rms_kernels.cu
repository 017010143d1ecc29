// Root-mean-square norm of rows on the caller's device tensors, with the addition of a residual stream and an output of 8 bits with scales.
//
//   forward    h = x + residual,  rstd = 1 / sqrt(sum(h^2) / n + eps),  y = h * rstd * weight
//   8 bits     s = max(max |y| over a group of columns / 448, 2^-126),  q = e4m3(y / s)
//   backward   xh = h * rstd,  t = dy * weight,  dx = rstd * (t - xh * mean(t * xh)) + dresidual,  dweight = sum over rows of dy * xh
//
// The norm is that of the 32-bit sum; the stream's h is rounded to the tensors' type for whoever reads it next.  All are bound by memory: 4 to 10 operations
// per element that is read and written once; a row stays in the registers of its threads.  Sums are fp32 in a fixed order: a thread's
// columns in ascending order, then halves of the lanes, then the warps in order.  A sum of squares that leaves fp32's range is taken again at a
// scale of 2^-100 or 2^100, which costs the rows that need it nothing but instructions.
//
// Measured (inputs not in L2): 65536 x 1536 bf16 with a residual 118 us (6.8 TB/s), its backward pass in fp32 with the residual's gradient 242 us (6.7 TB/s, 7 of them the columns' sums);
// 8 bits, 40000 x 1000 fp16 in groups of 128 25 us (4.9 TB/s: 430 instructions per row, issue slots at 64 %; 25.5 where rms is above 1).  16 x 1536: 1.8 us.
#include "rms.cuh"

namespace {

// Backward: a block of W warps per row (W = 1: rows side by side, L lanes each) takes R rows at a time, walks down the rows and keeps its columns' weight
// gradients in registers; part_w: [blocks][n] (of a single block the gradient itself), or NULL.
constexpr int rms_per_sm_back(int warps) { return warps == 1 ? 4 : 24 / warps < 1 ? 1 : 24 / warps; }

template <typename T, int W, int L, int VEC, int CH, int R>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32, rms_per_sm_back(W))
k_rms_backward(const T* dy, int64_t dy_stride, const T* h, int64_t h_stride, const float* rstd, const float* weight, const T* dres, int64_t dres_stride, int64_t rows, int n,
               T* dx, int64_t dx_stride, float* __restrict__ part_w) {
    constexpr int LANES = W == 1 ? L : 32 * W, SUBS = W == 1 ? 32 / L : 1, RB = W == 1 ? 4 * SUBS : 1;
    __shared__ float s_sum[2][R][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane % L : threadIdx.x;
    float w[CH][VEC], aw[CH][VEC];
    op_next_may_start();
    op_wait_for_previous();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LANES + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[c][i] = aw[c][i] = 0.0f;
        if (col < n) norm_columns<VEC>(weight, col, 1.0f, w[c]);
    }
    const float inv_n = 1.0f / (float)n;
    int turn = 0;
    // the lanes of a warp take the same number of turns
    for (int64_t turn0 = ((int64_t)blockIdx.x * RB + (W == 1 ? warp * SUBS : 0)) * R; turn0 < rows; turn0 += (int64_t)gridDim.x * RB * R, turn ^= 1) {
        const int64_t first = turn0 + (SUBS > 1 ? lane / L * R : 0);
        OpRaw<T, VEC> hv[R][CH], gv[R][CH], dv[R][CH];
        float r[R], s[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const bool in = first + q < rows;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LANES + t) * VEC;
                hv[q][c].zero();
                gv[q][c].zero();
                dv[q][c].zero();
                if (in && col < n) {
                    hv[q][c].load(h + (first + q) * h_stride + col);
                    gv[q][c].load(dy + (first + q) * dy_stride + col);
                    if (dres) dv[q][c].load(dres + (first + q) * dres_stride + col);
                }
            }
            r[q] = in ? rstd[first + q] : 0.0f;
        }
        // columns and rows that do not exist are zeros throughout
#pragma unroll
        for (int q = 0; q < R; ++q) {
            s[q] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = hv[q][c].get(i) * r[q], g = gv[q][c].get(i);
                    aw[c][i] = fmaf(g, xh, aw[c][i]);
                    s[q] = fmaf(g * w[c][i], xh, s[q]);
                }
        }
        if (W > 1) norm_block_sums<W, R>(s, reinterpret_cast<float(*)[R]>(s_sum[turn]), warp, lane);  // a warp that is a round ahead writes the other set
        else norm_rows_sum<1, L, R>(s, nullptr, warp, lane);
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const float m = s[q] * inv_n;
            if (first + q < rows)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LANES + t) * VEC;
                    if (col < n) {
                        float o[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) o[i] = fmaf(r[q], gv[q][c].get(i) * w[c][i] - hv[q][c].get(i) * r[q] * m, dv[q][c].get(i));
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
                for (int i = 0; i < VEC; ++i) aw[c][i] += __shfl_xor_sync(0xffffffffu, aw[c][i], o);
    if (W == 1) {  // the four warps' sums, in order
        __shared__ float s_acc[3][32 * CH * VEC];
        if (warp > 0)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s_acc[warp - 1][(c * VEC + i) * 32 + lane] = aw[c][i];
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) aw[c][i] += s_acc[q][(c * VEC + i) * 32 + lane];
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LANES + t) * VEC;
        if (col < n && (SUBS == 1 || lane < L)) op_store<float, VEC>(part_w + (int64_t)blockIdx.x * n + col, aw[c]);  // n is a multiple of VEC
    }
}

// rows longer than RMS_REG_N_BACK: dx by a block per row, the columns' sums by threads that walk down stripes of rows
template <typename T, typename C>
__global__ void __launch_bounds__(1024)
k_rms_backward_long(const T* dy, int64_t dy_stride, const T* h, int64_t h_stride, const float* rstd, const float* weight, const T* dres, int64_t dres_stride, int n, T* dx,
                    int64_t dx_stride) {
    __shared__ float s_sum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T *hr = h + row * h_stride, *gr = dy + row * dy_stride, *rr = dres + row * dres_stride;
    op_next_may_start();
    op_wait_for_previous();
    const float r = rstd[row];
    float s = 0.0f;
    for (C c = threadIdx.x; c < n; c += 1024) s = fmaf(op_float(gr[c]) * (weight ? weight[c] : 1.0f), op_float(hr[c]) * r, s);
    const float m = norm_row_sum<32>(s, s_sum, warp, lane) / (float)n;
    T* dr = dx + row * dx_stride;
    for (C c = threadIdx.x; c < n; c += 1024)
        dr[c] = op_round<T>(fmaf(r, op_float(gr[c]) * (weight ? weight[c] : 1.0f) - op_float(hr[c]) * r * m, dres ? op_float(rr[c]) : 0.0f));
}
template <typename T>
__global__ void __launch_bounds__(256)
k_rms_columns_long(const T* dy, int64_t dy_stride, const T* h, int64_t h_stride, const float* rstd, int64_t rows, int n, float* __restrict__ part_w) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;  // may be beyond 2^31
    op_next_may_start();
    op_wait_for_previous();
    if (at >= (unsigned)n) return;
    const int col = (int)at;
    float aw = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) aw = fmaf(op_float(dy[row * dy_stride + col]), op_float(h[row * h_stride + col]) * rstd[row], aw);
    part_w[(int64_t)blockIdx.y * n + col] = aw;
}

// Warps per row that walk down the rows: eight columns a thread up to 4096 columns (two rows at a time), sixteen above (one row).
int rms_warps_back(int n) { return n <= 4096 ? norm_warps(n) : n <= 8192 ? 16 : 32; }
// Blocks: at most what runs at once; 16 rows or more for each, or the blocks' rows of gradients cost as much as the rows themselves, but four per SM as far as the rows go (4096 x 1024
// fp32: 12.1 us, with one per SM 17.4; 1718 x 443 fp16 7.6 and 11.9).
int rms_backward_blocks(int64_t rows, int n) {
    if (n > RMS_REG_N_BACK) return (int)(rows < 64 ? (rows < 1 ? 1 : rows) : 64);
    const int w = rms_warps_back(n);
    const int64_t turn = n <= 64 ? 32 : n <= 128 ? 16 : w == 1 ? 8 : n <= 4096 ? 2 : 1, sms = sm_count(), most = sms * rms_per_sm_back(w);
    const int64_t turns = (rows + turn - 1) / turn, least = (16 + turn - 1) / turn, want = (turns + least - 1) / least;
    if (turns <= 2) return 1;  // no second launch then
    const int64_t spread = 4 * sms < most ? 4 * sms : most, few = turns < spread ? turns : spread;
    return (int)(want < few ? few : want < most ? want : most);
}

struct RmsBackward {
    cudaStream_t s;
    const void* dy;
    int64_t dys;
    const void* h;
    int64_t hs;
    const float *rstd, *w;
    const void* dres;
    int64_t drs;
    int64_t rows;
    int n;
    void* dx;
    int64_t dxs;
    float* part_w;
    int blocks;
};
template <typename T, int VEC, int W, int L, int K, int R>
void rms_backward_go(const RmsBackward& a) {
    op_launch_next(a.s, dim3((unsigned)a.blocks), dim3(W == 1 ? 128 : W * 32), 0, k_rms_backward<T, W, L, VEC, K / VEC, R>, (const T*)a.dy, a.dys, (const T*)a.h, a.hs, a.rstd, a.w, (const T*)a.dres, a.drs,
                   a.rows, a.n, (T*)a.dx, a.dxs, a.part_w);
}
template <typename T, int VEC>
void rms_backward_pick(const RmsBackward& a) {
    if (a.n > RMS_REG_N_BACK) {
        // the columns first: dx may be dy's or h's memory
        if (a.part_w)
            op_launch_next(a.s, dim3((unsigned)ceil_div64(a.n, 256), (unsigned)a.blocks), dim3(256), 0, k_rms_columns_long<T>, (const T*)a.dy, a.dys, (const T*)a.h, a.hs, a.rstd, a.rows, a.n, a.part_w);
        op_launch_next(a.s, dim3((unsigned)a.rows), dim3(1024), 0, a.n <= INT32_MAX - 1023 ? k_rms_backward_long<T, int> : k_rms_backward_long<T, int64_t>, (const T*)a.dy, a.dys, (const T*)a.h, a.hs, a.rstd,
                       a.w, (const T*)a.dres, a.drs, a.n, (T*)a.dx, a.dxs);
    } else if (a.n <= 64) {
        rms_backward_go<T, VEC, 1, 8, 8, 2>(a);
    } else if (a.n <= 128) {
        rms_backward_go<T, VEC, 1, 16, 8, 2>(a);
    } else if (a.n > 8192) {
        rms_backward_go<T, VEC, 32, 32, 16, 1>(a);
    } else if (a.n > 4096) {
        rms_backward_go<T, VEC, 16, 32, 16, 1>(a);
    } else {
        norm_with_warps<1>(norm_warps(a.n), [&](auto w) { rms_backward_go<T, VEC, decltype(w)::value, 32, 8, 2>(a); });
    }
}

#define RMS_MAX_ROWS 2147483647LL

// whether two tensors of the same shape are the same memory, element by element
bool rms_same(const void* a, int64_t as, const void* b, int64_t bs, int64_t rows) { return a == b && (as == bs || rows == 1); }

int rms_forward_check(const RmsForward& a, int type, bool eight, char* err, size_t err_len) {
    const int size = op_type_size(type);
    if (!size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (a.rows < 0 || a.rows > RMS_MAX_ROWS || a.n < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^31) and n positive");
    if (!(a.eps >= 0.0f)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "eps must not be negative");
    if (eight && a.group != 32 && a.group != 64 && a.group != 128 && a.group != a.n) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "group must be 32, 64, 128 or n (got %d)", a.group);
    if (a.h && !a.r) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_h needs a residual: without one it would be x");
    if (a.rows == 0) return TB_OK;
    if (!a.x || !a.y || (eight && !a.scale)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (a.rows > 1 && (a.xs < a.n || a.ys < a.n || (a.r && a.rs < a.n) || (a.h && a.hs < a.n))) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if (((uintptr_t)a.x | (uintptr_t)a.r | (uintptr_t)a.h | (eight ? 0 : (uintptr_t)a.y)) % size || ((uintptr_t)a.w | (uintptr_t)a.rstd | (uintptr_t)a.scale) & 3)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const int64_t row = (int64_t)a.n * size, groups = eight ? (a.n + (int64_t)a.group - 1) / a.group : 0;
    const OpRows xr = {a.x, a.xs * size, a.rows, row}, rr = {a.r, a.rs * size, a.rows, row}, hr = {a.h, a.hs * size, a.rows, row};
    const OpRows yr = {a.y, eight ? a.ys : a.ys * size, a.rows, eight ? a.n : row};
    const OpRows wv = op_vector(a.w, a.n), dv = op_vector(a.rstd, a.rows), sv = op_vector(a.scale, a.rows * groups);
    const auto apart = [&](const void* in, int64_t is, const void* out, int64_t os) { return !in || !out || op_apart(in, 0, is, out, 0, os, 1, a.rows, a.n, size); };
    if (!apart(a.x, a.xs, a.h, a.hs) || !apart(a.r, a.rs, a.h, a.hs)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_h overlaps d_x or d_residual in part");
    if (eight ? op_extents_meet(yr, {xr, rr, hr})
              : !apart(a.x, a.xs, a.y, a.ys) || !apart(a.r, a.rs, a.y, a.ys) || !apart(a.h, a.hs, a.y, a.ys) || (a.h && rms_same(a.h, a.hs, a.y, a.ys, a.rows)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "%s overlaps another tensor", eight ? "d_q" : "d_y");
    if (op_meets(yr, {wv, dv, sv}) || op_meets(hr, {wv, dv, sv}) || op_meets(xr, {dv, sv}) || op_meets(rr, {dv, sv}) || op_meets(wv, {dv, sv}) || op_meets(dv, {sv}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    return TB_OK;
}
int rms_forward_run(const RmsForward& a, int type, char* err, size_t err_len) {
    const int size = op_type_size(type), vec = 16 / size;
    const bool out = a.group ? (uintptr_t)a.y % vec == 0 && a.ys % vec == 0 : norm_aligned(a.y, a.ys, size);
    const bool wide = a.n % vec == 0 && norm_aligned(a.x, a.xs, size) && (!a.r || norm_aligned(a.r, a.rs, size)) && (!a.h || norm_aligned(a.h, a.hs, size)) && out && (uintptr_t)a.w % (4 * vec) == 0;
    if (a.group) rms_quantised_run(a, type, wide);
    else if (type == TB_TYPE_F32) wide ? rms_forward_pick<float, 4, 0>(a) : rms_forward_pick<float, 1, 0>(a);
    else if (type == TB_TYPE_F16) wide ? rms_forward_pick<__half, 8, 0>(a) : rms_forward_pick<__half, 1, 0>(a);
    else wide ? rms_forward_pick<__nv_bfloat16, 8, 0>(a) : rms_forward_pick<__nv_bfloat16, 1, 0>(a);
    return op_launched(err, err_len);
}

}  // namespace

extern "C" int tb_rms_norm_forward(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const float* d_weight, float eps, int type, int64_t rows, int n, void* d_y,
                                   int64_t y_stride, void* d_h, int64_t h_stride, float* d_rstd, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const RmsForward a = {static_cast<cudaStream_t>(stream), d_x, x_stride, d_residual, residual_stride, d_weight, eps, rows, n, d_y, y_stride, d_h, h_stride, d_rstd, nullptr, 0};
    const int rc = rms_forward_check(a, type, false, err, err_len);
    return rc != TB_OK || rows == 0 ? rc : rms_forward_run(a, type, err, err_len);
}

extern "C" int tb_rms_norm_quantised(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const float* d_weight, float eps, int type, int64_t rows, int n, int group,
                                     void* d_q, int64_t q_stride, float* d_scale, void* d_h, int64_t h_stride, float* d_rstd, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const RmsForward a = {static_cast<cudaStream_t>(stream), d_x, x_stride, d_residual, residual_stride, d_weight, eps, rows, n, d_q, q_stride, d_h, h_stride, d_rstd, d_scale, group};
    const int rc = rms_forward_check(a, type, true, err, err_len);
    return rc != TB_OK || rows == 0 ? rc : rms_forward_run(a, type, err, err_len);
}

extern "C" int64_t tb_rms_norm_backward_workspace(int64_t rows, int n) {
    if (rows < 0 || rows > RMS_MAX_ROWS || n < 1) return TB_ERR_INVALID_ARGUMENT;
    return (int64_t)rms_backward_blocks(rows, n) * n * (int64_t)sizeof(float);
}

extern "C" int tb_rms_norm_backward(const void* d_dy, int64_t dy_stride, const void* d_h, int64_t h_stride, const float* d_rstd, const float* d_weight, const void* d_dresidual, int64_t dresidual_stride,
                                    int type, int64_t rows, int n, void* d_dx, int64_t dx_stride, float* d_dweight, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int size = op_type_size(type);
    if (!size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (rows < 0 || rows > RMS_MAX_ROWS || n < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^31) and n positive");
    if (rows > 0 && (!d_dy || !d_h || !d_rstd || !d_dx)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (rows > 1 && (dy_stride < n || h_stride < n || dx_stride < n || (d_dresidual && dresidual_stride < n))) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if (((uintptr_t)d_dy | (uintptr_t)d_h | (uintptr_t)d_dx | (uintptr_t)d_dresidual) % size || ((uintptr_t)d_weight | (uintptr_t)d_rstd | (uintptr_t)d_dweight) & 3)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const auto apart = [&](const void* in, int64_t is) { return !in || op_apart(in, 0, is, d_dx, 0, dx_stride, 1, rows, n, size); };
    if (rows > 0 && (!apart(d_dy, dy_stride) || !apart(d_h, h_stride) || !apart(d_dresidual, dresidual_stride)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dx overlaps d_dy, d_h or d_dresidual in part");
    const int64_t need = tb_rms_norm_backward_workspace(rows, n);
    if (d_dweight && (!d_work || work_bytes < need || ((uintptr_t)d_work & 31)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    const int64_t row = (int64_t)n * size;
    const OpRows wv = op_vector(d_weight, n), rv = op_vector(d_rstd, rows), dwv = op_vector(d_dweight, n);
    const OpRows gr = {d_dy, dy_stride * size, rows, row}, hr = {d_h, h_stride * size, rows, row}, sr = {d_dresidual, dresidual_stride * size, rows, row}, dr = {d_dx, dx_stride * size, rows, row};
    if (rows > 0 && (op_meets(dr, {wv, rv, dwv}) || op_meets(gr, {dwv}) || op_meets(hr, {dwv}) || op_meets(sr, {dwv}) || op_meets(wv, {dwv}) || op_meets(rv, {dwv})))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (d_dweight) op_note(cudaMemsetAsync(d_dweight, 0, (size_t)n * sizeof(float), s));
        return op_launched(err, err_len);
    }
    const int blocks = rms_backward_blocks(rows, n);
    const bool wide = n % (16 / size) == 0 && norm_aligned(d_dy, dy_stride, size) && norm_aligned(d_h, h_stride, size) && norm_aligned(d_dx, dx_stride, size) &&
                      (!d_dresidual || norm_aligned(d_dresidual, dresidual_stride, size)) && ((uintptr_t)d_weight & 15) == 0;
    // a single block writes the gradient itself (its stores are as wide as 32 bytes)
    const bool direct = blocks == 1 && d_dweight && ((uintptr_t)d_dweight & 31) == 0;
    const RmsBackward a = {s, d_dy, dy_stride, d_h, h_stride, d_rstd, d_weight, d_dresidual, dresidual_stride, rows, n, d_dx, dx_stride, direct ? d_dweight : d_dweight ? static_cast<float*>(d_work) : nullptr, blocks};
    if (type == TB_TYPE_F32) wide ? rms_backward_pick<float, 4>(a) : rms_backward_pick<float, 1>(a);
    else if (type == TB_TYPE_F16) wide ? rms_backward_pick<__half, 8>(a) : rms_backward_pick<__half, 1>(a);
    else wide ? rms_backward_pick<__nv_bfloat16, 8>(a) : rms_backward_pick<__nv_bfloat16, 1>(a);
    if (d_dweight && !direct) op_launch_next(s, dim3((unsigned)ceil_div64(n, 8), 1), dim3(1024), 0, k_norm_columns_final, (const float*)d_work, blocks, n, d_dweight, (float*)nullptr);
    return op_launched(err, err_len);
}
