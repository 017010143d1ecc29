// Newton-Schulz orthogonalisation of matrices with a short side of up to 64 (the hidden layers of a net) and the entry points of
// both paths.
//
// Short side n <= 64.  X after the steps is P(G) U with a polynomial P of the Gram matrix G = U U^T alone, so the long side is read
// twice and the steps run on n x n matrices:
//   G = U U^T (its trace is |U|^2, so no pass for the norm), A = G / (|U| + eps)^2, P = I;
//   steps times: Q = a I + b A + c A^2, P = Q P, A = (Q A) Q;   out = P U / (|U| + eps)
// The Gram matrix squares the singular values and P grows like a^steps towards the small ones, so all of this is 64-bit: a
// singular value 1e-3 of the largest would lose 1e-2 of itself with fp32 sums, here nothing is lost.  What bounds it is latency: a cluster
// of CTAs shares the long side of a matrix, every CTA adds up the CTAs' Gram matrices (distributed shared memory, in order) and
// runs the steps by itself, which costs less than telling the others.  All matrices are polynomials of one symmetric matrix, so they are
// symmetric and commute: half of every product is computed.  A fixed order everywhere: results repeat bit for bit.
#include "orth.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

#define SMALL_THREADS 256
#define SMALL_CHUNK 4096  // doubles of a chunk of columns in shared memory

// TS x TS entries of a symmetric product per thread; pitch: of the matrices' rows
template <int TS>
__device__ __forceinline__ void small_product(const double* __restrict__ x, const double* __restrict__ y, double* __restrict__ out, int np, int pitch, int ti, int tj,
                                              double scale, double ident, const double* __restrict__ add, double add_scale) {
    double acc[TS][TS];
#pragma unroll
    for (int r = 0; r < TS; ++r)
#pragma unroll
        for (int c = 0; c < TS; ++c) acc[r][c] = 0.0;
    if (ti >= 0) {
#pragma unroll 4
        for (int k = 0; k < np; ++k) {
            double a[TS], b[TS];
#pragma unroll
            for (int r = 0; r < TS; ++r) a[r] = x[k * pitch + ti * TS + r];
#pragma unroll
            for (int c = 0; c < TS; ++c) b[c] = y[k * pitch + tj * TS + c];
#pragma unroll
            for (int r = 0; r < TS; ++r)
#pragma unroll
                for (int c = 0; c < TS; ++c) acc[r][c] = fma(a[r], b[c], acc[r][c]);
        }
#pragma unroll
        for (int r = 0; r < TS; ++r)
#pragma unroll
            for (int c = 0; c < TS; ++c) {
                const int i = ti * TS + r, j = tj * TS + c;
                double v = acc[r][c] * scale;
                if (add) v = fma(add_scale, add[i * pitch + j], v);
                if (i == j) v += ident;
                out[i * pitch + j] = v;
                out[j * pitch + i] = v;
            }
    }
}

// the lower triangle's tile of a linear index: t = ti (ti + 1) / 2 + tj
__device__ __forceinline__ void small_tile(int t, int& ti, int& tj) {
    ti = 0;
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = t - ti * (ti + 1) / 2;
}

// columns [j0, j0 + jc) of a matrix into xs[j][pitch] (64 bits); rows n .. np - 1 are zero
template <typename T, bool FIRST>
__device__ __forceinline__ void small_fill(const OrthIo& io, int b, int n, int np, bool tall, int64_t j0, int jc, double* xs, int pitch) {
    for (int e = threadIdx.x; e < np * jc; e += SMALL_THREADS) {
        // neighbours in memory go to neighbouring threads
        const int i = tall ? e % np : e / jc, j = tall ? e / np : e % jc;
        double v = 0.0;
        if (i < n) v = (double)(tall ? orth_load<T, FIRST>(io, b, j0 + j, i) : orth_load<T, FIRST>(io, b, i, j0 + j));
        xs[j * pitch + i] = v;
    }
}

// TS: side of a thread's part of the n x n products
template <typename T, int TS>
__global__ void __launch_bounds__(SMALL_THREADS) k_orth_small(OrthIo io, OrthPoly poly) {
    extern __shared__ double s_mem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.y, tid = threadIdx.x;
    const bool tall = io.rows > io.cols;
    const int n = tall ? io.cols : io.rows;
    const int64_t m = tall ? io.rows : io.cols;
    const int np = (n + 3) / 4 * 4, pitch = np + 2;  // rows of matrices start two banks apart
    const int xp = np + 1;                           // pitch of the columns' chunk
    const int jc_max = SMALL_CHUNK / np;
    double* s_x = s_mem;                            // [jc_max][xp], also the partial sums
    double* s_own = s_x + SMALL_CHUNK + jc_max;     // this CTA's Gram matrix, read by the others
    double* s_a = s_own + np * pitch;
    double* s_q = s_a + np * pitch;
    double* s_p = s_q + np * pitch;
    double* s_t = s_p + np * pitch;
    const int64_t per = (m + cs - 1) / cs, begin = min(m, per * rank), end = min(m, begin + per);

    // Gram matrix of this CTA's columns: 4 x 4 entries per thread, the columns of a chunk dealt to `groups` threads per tile
    const int tiles4 = (np / 4) * (np / 4 + 1) / 2, groups = min(SMALL_THREADS / tiles4, 32);
    const int t4 = tid % tiles4, kg = tid / tiles4;
    int gi, gj;
    small_tile(t4, gi, gj);
    double acc[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = 0.0;
    for (int64_t j0 = begin; j0 < end; j0 += jc_max) {
        const int jc = (int)min((int64_t)jc_max, end - j0);
        __syncthreads();
        small_fill<T, true>(io, b, n, np, tall, j0, jc, s_x, xp);
        __syncthreads();
        if (kg < groups)
            for (int j = kg; j < jc; j += groups) {
                double x[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = s_x[j * xp + gi * 4 + r];
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = s_x[j * xp + gj * 4 + c];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[r][c] = fma(x[r], y[c], acc[r][c]);
            }
    }
    __syncthreads();
    if (kg < groups)
#pragma unroll
        for (int e = 0; e < 16; ++e) s_x[(e * groups + kg) * tiles4 + t4] = acc[e / 4][e % 4];
    __syncthreads();
    for (int e = tid; e < 16 * tiles4; e += SMALL_THREADS) {
        const int t = e % tiles4, q = e / tiles4;
        double v = 0.0;
        for (int k = 0; k < groups; ++k) v += s_x[(q * groups + k) * tiles4 + t];
        int ti, tj;
        small_tile(t, ti, tj);
        const int i = ti * 4 + q / 4, j = tj * 4 + q % 4;
        s_own[i * pitch + j] = v;
        s_own[j * pitch + i] = v;
    }
    cluster.sync();
    for (int e = tid; e < np * np; e += SMALL_THREADS) {
        const int at = (e / np) * pitch + e % np;
        double v = 0.0;
        for (int r = 0; r < cs; ++r) v += cluster.map_shared_rank(s_own, r)[at];
        s_a[at] = v;
    }
    cluster.sync();  // nobody leaves, or reads on, while another reads its part
    __shared__ double s_inv;
    if (tid == 0) {
        double trace = 0.0;
        for (int i = 0; i < n; ++i) trace += s_a[i * pitch + i];
        s_inv = 1.0 / (sqrt(trace) + (double)poly.eps);
    }
    __syncthreads();
    const double inv = s_inv;
    // a matrix of zeros with eps 0: 0 / 0, as the definition says
    for (int e = tid; e < np * np; e += SMALL_THREADS) {
        const int at = (e / np) * pitch + e % np;
        s_a[at] = s_a[at] * inv * inv;
    }
    __syncthreads();

    const int tiles = (np / TS) * (np / TS + 1) / 2;
    int ti = -1, tj = 0;
    if (tid < tiles) small_tile(tid, ti, tj);
    for (int s = 0; s < poly.steps; ++s) {
        const bool last = s + 1 == poly.steps;
        small_product<TS>(s_a, s_a, s_q, np, pitch, ti, tj, poly.c, poly.a, s_a, poly.b);  // Q
        __syncthreads();
        // P = Q P (P = Q in the first step) and, unless it is the last, A = (Q A) Q
        if (s == 0) {
            for (int e = tid; e < np * pitch; e += SMALL_THREADS) s_p[e] = s_q[e];
        } else {
            small_product<TS>(s_q, s_p, s_own, np, pitch, ti, tj, 1.0, 0.0, nullptr, 0.0);
        }
        if (!last) small_product<TS>(s_q, s_a, s_t, np, pitch, ti, tj, 1.0, 0.0, nullptr, 0.0);
        __syncthreads();
        if (s > 0) {
            double* z = s_p;
            s_p = s_own;
            s_own = z;
        }
        if (!last) {
            small_product<TS>(s_t, s_q, s_a, np, pitch, ti, tj, 1.0, 0.0, nullptr, 0.0);
            __syncthreads();
        }
    }

    // out = P U / (|U| + eps): 4 rows and 4 columns (a quarter of the chunk apart) per thread
    const int row_tiles = np / 4;
    for (int64_t j0 = begin; j0 < end; j0 += jc_max) {
        const int jc = (int)min((int64_t)jc_max, end - j0), quarter = (jc + 3) / 4;
        __syncthreads();
        small_fill<T, false>(io, b, n, np, tall, j0, jc, s_x, xp);
        __syncthreads();
        for (int t = tid; t < row_tiles * quarter; t += SMALL_THREADS) {
            const int it = tall ? t % row_tiles : t / quarter, jt = tall ? t / row_tiles : t % quarter;
            double o[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[r][c] = 0.0;
            for (int k = 0; k < n; ++k) {
                double p[4], x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = s_p[k * pitch + it * 4 + r];
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] = s_x[min(jt + c * quarter, jc - 1) * xp + k];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[r][c] = fma(p[r], x[c], o[r][c]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = jt + c * quarter;
                if (j >= jc) continue;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = it * 4 + r;
                    if (i >= n) continue;
                    const float v = (float)(o[r][c] * inv);
                    if (tall) orth_store<T>(io, b, j0 + j, i, v); else orth_store<T>(io, b, i, j0 + j, v);
                }
            }
        }
    }
}

template <typename T, int TS>
void orth_small_go(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int cs) {
    const int n = io.rows < io.cols ? io.rows : io.cols, np = (n + 3) / 4 * 4;
    const size_t smem = (size_t)(SMALL_CHUNK + SMALL_CHUNK / np + 5 * np * (np + 2)) * sizeof(double);
    cudaFuncSetAttribute(k_orth_small<T, TS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cs, (unsigned)io.batch);
    cfg.blockDim = dim3(SMALL_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, k_orth_small<T, TS>, io, p);
}
template <typename T>
void orth_small_pick(cudaStream_t s, const OrthIo& io, const OrthPoly& p) {
    const int n = io.rows < io.cols ? io.rows : io.cols, m = io.rows < io.cols ? io.cols : io.rows;
    int cs = 1;  // about 64 columns or more per CTA
    while (cs < 8 && cs * 64 < m) cs *= 2;
    if (n <= 16) orth_small_go<T, 1>(s, io, p, cs);
    else if (n <= 32) orth_small_go<T, 2>(s, io, p, cs);
    else orth_small_go<T, 4>(s, io, p, cs);
}

// The limbs hold numbers up to 32 (orth_tc.cu); fp16 inputs' results are rounded to 11 bits, bf16's to 8: one limb of 11 bits is
// enough for the latter.
int orth_limbs(int type) { return type == TB_TYPE_BF16 ? 1 : 2; }

// Singular values start at or below 1.  Whether the polynomial keeps them, Q and A inside what a limb holds.
bool orth_bounded(const OrthPoly& p) {
    double u = 1.0;
    for (int s = 0; s < p.steps; ++s) {
        const double lam = u * u;
        if (!(fabs((double)p.a) + fabs((double)p.b) * lam + fabs((double)p.c) * lam * lam <= 31.0)) return false;
        // extremes of a x + b x^3 + c x^5 on [0, u]
        double best = fabs(u * (p.a + p.b * lam + p.c * lam * lam));
        const double qa = 5.0 * p.c, qb = 3.0 * p.b, qc = p.a, disc = qb * qb - 4.0 * qa * qc;
        double roots[2] = {-1.0, -1.0};
        if (qa != 0.0 && disc >= 0.0) {
            roots[0] = (-qb + sqrt(disc)) / (2.0 * qa);
            roots[1] = (-qb - sqrt(disc)) / (2.0 * qa);
        } else if (qa == 0.0 && qb != 0.0) {
            roots[0] = -qc / qb;
        }
        for (double l : roots)
            if (l > 0.0 && l < lam) best = fmax(best, fabs(sqrt(l) * (p.a + p.b * l + p.c * l * l)));
        u = best;
        if (!(u <= 4.0)) return false;
    }
    return true;
}

int orth_check(int type, int batch, int rows, int cols, const OrthPoly& p, char* err, size_t err_len) {
    if (!op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (batch < 0 || batch > 65535 || rows < 1 || cols < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "batch must be in [0, 65535], rows and cols positive");
    if (p.steps < 1 || p.steps > 32) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "steps must be in [1, 32] (got %d)", p.steps);
    if (!(p.eps >= 0.0f)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "eps must not be negative");
    if (!orth_bounded(p)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "with these coefficients singular values could grow beyond 4, or the factors beyond 31");
    return TB_OK;
}

int64_t orth_workspace(int limbs, int batch, int rows, int cols) {
    return (rows < cols ? rows : cols) <= ORTH_SMALL_N ? 0 : orth_tc_workspace(batch, rows, cols, limbs);
}

int orth_run(const OrthIo& io, const OrthPoly& p, int type, int limbs, void* work, int64_t work_bytes, cudaStream_t s, char* err, size_t err_len) {
    const int64_t need = orth_workspace(limbs, io.batch, io.rows, io.cols);
    if (need > 0 && (!work || work_bytes < need || ((uintptr_t)work & 127)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be 128-byte aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    if ((io.rows < io.cols ? io.rows : io.cols) <= ORTH_SMALL_N) launch_orth_small(s, io, p, type);
    else launch_orth_tc(s, io, p, type, limbs, work);
    return op_launched(err, err_len);
}

}  // namespace

void launch_orth_small(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int type) {
    if (type == TB_TYPE_F32) orth_small_pick<float>(s, io, p);
    else if (type == TB_TYPE_F16) orth_small_pick<__half>(s, io, p);
    else orth_small_pick<__nv_bfloat16>(s, io, p);
}

extern "C" int64_t tb_orthogonalise_workspace(int type, int batch, int rows, int cols) {
    if (!op_type_size(type) || batch < 0 || batch > 65535 || rows < 1 || cols < 1) return TB_ERR_INVALID_ARGUMENT;
    return orth_workspace(orth_limbs(type), batch, rows, cols);
}

extern "C" int tb_orthogonalise(const void* d_x, int64_t x_batch, int64_t x_stride, int type, int batch, int rows, int cols, int steps, const float* coefficients,
                                float eps, void* d_out, int64_t out_batch, int64_t out_stride, void* d_work, int64_t work_bytes, void* stream, char* err,
                                size_t err_len) {
    if (err && err_len) err[0] = 0;
    if (!coefficients) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "coefficients is NULL");
    const OrthPoly p = {steps, coefficients[0], coefficients[1], coefficients[2], eps};
    const int rc = orth_check(type, batch, rows, cols, p, err, err_len);
    if (rc != TB_OK) return rc;
    if (batch == 0) return TB_OK;
    if (!d_x || !d_out) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_x or d_out is NULL");
    if (((uintptr_t)d_x | (uintptr_t)d_out) % op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_x and d_out must be aligned to their elements");
    if (rows > 1 && (x_stride < cols || out_stride < cols)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least cols");
    if (batch > 1 && (x_batch < (rows - 1) * x_stride + cols || out_batch < (rows - 1) * out_stride + cols))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "matrices of the batch overlap");
    OrthIo io = {};
    io.g = d_x;
    io.g_batch = x_batch;
    io.g_stride = x_stride;
    io.out = d_out;
    io.out_batch = out_batch;
    io.out_stride = out_stride;
    io.rows = rows;
    io.cols = cols;
    io.batch = batch;
    return orth_run(io, p, type, orth_limbs(type), d_work, work_bytes, static_cast<cudaStream_t>(stream), err, err_len);
}

extern "C" int64_t tb_muon_step_workspace(int batch, int rows, int cols) {
    if (batch < 0 || batch > 65535 || rows < 1 || cols < 1) return TB_ERR_INVALID_ARGUMENT;
    return orth_workspace(2, batch, rows, cols);
}

extern "C" int tb_muon_step(const tb_muon* cfg, const float* d_w, const float* d_m, const void* d_g, int g_type, int batch, int rows, int cols, float* d_w_out,
                            float* d_m_out, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    if (!cfg || cfg->struct_size != (int32_t)sizeof(tb_muon)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tb_muon is NULL or of another size");
    const OrthPoly p = {cfg->steps, cfg->a, cfg->b, cfg->c, cfg->eps};
    const int rc = orth_check(g_type, batch, rows, cols, p, err, err_len);
    if (rc != TB_OK) return rc;
    if (!(cfg->clip > 0.0f)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "clip must be positive (INFINITY: none)");
    if (batch == 0) return TB_OK;
    if (!d_w || !d_m || !d_g || !d_w_out || !d_m_out) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (((uintptr_t)d_w | (uintptr_t)d_m | (uintptr_t)d_w_out | (uintptr_t)d_m_out) & 3 || (uintptr_t)d_g % op_type_size(g_type))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    OrthIo io = {};
    io.g = d_g;
    io.g_batch = io.out_batch = (int64_t)rows * cols;
    io.g_stride = io.out_stride = cols;
    io.m = d_m;
    io.m_out = d_m_out;
    io.beta = cfg->beta;
    io.nesterov = cfg->nesterov;
    io.out = d_w_out;
    io.w = d_w;
    io.w_mul = (float)(1.0 - (double)cfg->lr * (double)cfg->weight_decay);
    io.step = (float)((double)cfg->lr * (double)cfg->scale);
    io.clip = cfg->clip;
    io.rows = rows;
    io.cols = cols;
    io.batch = batch;
    return orth_run(io, p, g_type, 2, d_work, work_bytes, static_cast<cudaStream_t>(stream), err, err_len);
}
