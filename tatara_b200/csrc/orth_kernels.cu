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
// symmetric and commute: half of every product is computed.  The products are the tensor cores' 64-bit ones (8 x 8 x 4 per warp): a step of
// 32 x 32 matrices waits for a chain of four of them where thread-wise sums wait for sixteen additions and four times the shared-memory
// reads.  A fixed order everywhere: results repeat bit for bit.
// Measured: 9 matrices of 16 x 1536 11.9 us (the loads 2.4, the steps 4), the Muon step of 1024 x 32 15.6 us (the steps 7), 64 x 512 43.7 us (the steps 36:
// 64-bit products at 40 of the 64 multiply-adds per cycle and SM).
#include "orth.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace cg = cooperative_groups;

namespace {

#define SMALL_CLUSTER 16   // most CTAs that share a matrix
#define SMALL_SMEM 229376  // 224 KB
#define SMALL_BATCH 8      // elements a thread has on their way at once

// rows of 64-bit matrices start 4 doubles apart modulo 16: the 4 x 8 operands below touch every bank once
__host__ __device__ constexpr int small_pitch(int np) { return (np + 11) / 16 * 16 + 4; }

// C (8 x 8) += A (8 x 4) B (4 x 8) in 64 bits; lane l holds A[l / 4][l % 4], B[l % 4][l / 4], C[l / 4][2 (l % 4) + {0, 1}]
__device__ __forceinline__ void small_mma(double (&c)[2], double a, double b) {
    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// the lower triangle's block of a linear index: t = bi (bi + 1) / 2 + bj
__device__ __forceinline__ void small_block(int t, int& bi, int& bj) {
    bi = 0;
    while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
    bj = t - bi * (bi + 1) / 2;
}

// Block (bi, bj) of out = x y or, with LINEAR, scale x y + linear x + ident I, by one warp, and its mirror image: the matrices are symmetric and
// commute.  Two chains; what does not depend on them is ready when they are (a 64-bit addition takes as long as a quarter of the chain).
template <bool LINEAR>
__device__ __forceinline__ void small_product(const double* __restrict__ x, const double* __restrict__ y, double* __restrict__ out, int np, int pitch, int block, int lane,
                                              double scale, double linear, double ident) {
    const int bi = block >> 8, bj = block & 255, i = bi * 8 + (lane >> 2), j = bj * 8 + 2 * (lane & 3);
    const double *a = x + (lane & 3) * pitch + i, *b = y + (lane & 3) * pitch + bj * 8 + (lane >> 2);
    double c[2][2] = {{0.0, 0.0}, {0.0, 0.0}}, rest[2] = {0.0, 0.0};
    if (LINEAR)
#pragma unroll
        for (int q = 0; q < 2; ++q) rest[q] = fma(linear, x[i * pitch + j + q], i == j + q ? ident : 0.0);
#pragma unroll 4
    for (int k = 0; k < np; k += 8, a += 8 * pitch, b += 8 * pitch) {
        small_mma(c[0], a[0], b[0]);
        small_mma(c[1], a[4 * pitch], b[4 * pitch]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const double v = LINEAR ? fma(scale, c[0][q], fma(scale, c[1][q], rest[q])) : c[0][q] + c[1][q];
        if (i >= j + q) {
            out[i * pitch + j + q] = v;
            out[(j + q) * pitch + i] = v;
        }
    }
}

// columns [j0, j0 + jc) of a matrix into xs[j][pitch] (64 bits); rows n .. np - 1 and columns jc .. jp - 1 are zero.  Neighbours in memory go to
// neighbouring threads; all loads of a batch are issued before the first is used (one at a time this was half of the kernel).
template <typename T, bool FIRST, int THREADS>
__device__ __forceinline__ void small_fill(const OrthIo& io, int b, int n, int np, bool tall, int64_t j0, int jc, int jp, double* xs, int pitch) {
    const int total = np * jp, inner = tall ? np : jp;
    const unsigned magic = (unsigned)((0x100000000ull + inner - 1) / inner);  // e / inner = e * magic >> 32 for e * inner < 2^32
    for (int e0 = threadIdx.x; e0 < total; e0 += THREADS * SMALL_BATCH) {
        float g[SMALL_BATCH], m[SMALL_BATCH];
        int64_t at[SMALL_BATCH];
        int to[SMALL_BATCH];
#pragma unroll
        for (int u = 0; u < SMALL_BATCH; ++u) {
            const int e = e0 + u * THREADS;
            const int hi = (int)__umulhi((unsigned)e, magic), lo = e - hi * inner;
            const int i = tall ? lo : hi, j = tall ? hi : lo;
            to[u] = e < total ? j * pitch + i : -1;
            at[u] = -1;
            g[u] = m[u] = 0.0f;
            if (e < total && i < n && j < jc) {
                const int64_t r = tall ? j0 + j : i, c = tall ? i : j0 + j;
                g[u] = op_float(static_cast<const T*>(io.g)[b * io.g_batch + r * io.g_stride + c]);
                if (io.m) {
                    at[u] = ((int64_t)b * io.rows + r) * io.cols + c;
                    m[u] = FIRST ? io.m[at[u]] : io.m_out[at[u]];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < SMALL_BATCH; ++u) {
            float v = g[u];
            if (at[u] >= 0) {
                if (FIRST) {
                    m[u] = fmaf(io.beta, m[u], g[u]);
                    io.m_out[at[u]] = m[u];
                }
                v = io.nesterov ? fmaf(io.beta, m[u], g[u]) : m[u];
            }
            if (to[u] >= 0) xs[to[u]] = (double)v;
        }
    }
}

// jc_max: columns of a chunk in shared memory, a multiple of 8
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) k_orth_small(OrthIo io, OrthPoly poly, int jc_max) {
    constexpr int THREADS = 32 * WARPS;
    extern __shared__ double s_mem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool tall = io.rows > io.cols;
    const int n = tall ? io.cols : io.rows;
    const int64_t m = tall ? io.rows : io.cols;
    const int np = (n + 7) / 8 * 8, pitch = small_pitch(np), size = np * pitch, side = np / 8, blocks = side * (side + 1) / 2;
    double* s_x = s_mem;                     // [jc_max][pitch]
    double* s_own = s_x + jc_max * pitch;    // this CTA's Gram matrix by blocks [blocks][64], read by the others
    double* s_a = s_own + size;
    double* s_q = s_a + size;
    double* s_p = s_q + size;
    double* s_t = s_p + size;
    double* s_part = s_q;                    // partial sums of the Gram matrix
    const int64_t per = (m + cs - 1) / cs, begin = min(m, per * rank), end = min(m, begin + per);

    op_next_may_start();
    op_wait_for_previous();
    __shared__ int s_block[36];  // (bi, bj) of the lower triangle's blocks
    if (tid < blocks) {
        int bi, bj;
        small_block(tid, bi, bj);
        s_block[tid] = bi << 8 | bj;
    }
    // Gram matrix of this CTA's columns: a warp per block, or a few per block that share the columns
    const int splits = blocks < WARPS ? max(1, min(WARPS / blocks, jc_max / 8)) : 1, units = blocks * splits;
    constexpr int UNITS = 36 / WARPS + 1;  // of a warp: warp, warp + WARPS, ..
    double gram[UNITS][2];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) gram[u][0] = gram[u][1] = 0.0;
    for (int64_t j0 = begin; j0 < end; j0 += jc_max) {
        const int jc = (int)min((int64_t)jc_max, end - j0), jp = (jc + 7) / 8 * 8;
        if (j0 > begin) __syncthreads();
        small_fill<T, true, THREADS>(io, b, n, np, tall, j0, jc, jp, s_x, pitch);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int unit = warp + u * WARPS;
            if (unit >= units) break;
            const int bi = s_block[unit % blocks] >> 8, bj = s_block[unit % blocks] & 255;
            const double *x = s_x + (lane & 3) * pitch + bi * 8 + (lane >> 2), *y = s_x + (lane & 3) * pitch + bj * 8 + (lane >> 2);
#pragma unroll 4
            for (int j = unit / blocks * 4; j < jp; j += 4 * splits) small_mma(gram[u], x[j * pitch], y[j * pitch]);
        }
    }
    double* gram_to = splits > 1 ? s_part : s_own;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int unit = warp + u * WARPS;
        if (unit < units) *reinterpret_cast<double2*>(gram_to + unit * 64 + lane * 2) = make_double2(gram[u][0], gram[u][1]);
    }
    if (splits > 1) {
        __syncthreads();
        for (int e = tid; e < blocks * 64; e += THREADS) {
            double v = 0.0;
#pragma unroll
            for (int k = 0; k < WARPS; ++k)
                if (k < splits) v += s_part[k * blocks * 64 + e];
            s_own[e] = v;
        }
    }
    if (cs > 1) cluster.sync();
    else __syncthreads();
    // every CTA adds up its share of the entries over the CTAs, in order, and hands the sums to all
    for (int e = blocks * 32 * rank / cs + tid; e < blocks * 32 * (rank + 1) / cs; e += THREADS) {
        double2 part[SMALL_CLUSTER], v = make_double2(0.0, 0.0);
#pragma unroll
        for (int r = 0; r < SMALL_CLUSTER; ++r) part[r] = r < cs ? reinterpret_cast<const double2*>(cluster.map_shared_rank(s_own, r))[e] : make_double2(0.0, 0.0);
#pragma unroll
        for (int r = 0; r < SMALL_CLUSTER; ++r) {
            v.x += part[r].x;
            v.y += part[r].y;
        }
        for (int r = 0; r < cs; ++r) reinterpret_cast<double2*>(cluster.map_shared_rank(s_t, r))[e] = v;
    }
    if (cs > 1) cluster.sync();  // from here on no CTA touches another's memory
    else __syncthreads();
    double trace = 0.0;
    for (int i = lane; i < np; i += 32) {
        const int bi = i >> 3;
        trace += s_t[(bi * (bi + 1) / 2 + bi) * 64 + (i & 7) * 9];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) trace += __shfl_xor_sync(0xffffffffu, trace, o);
    // a matrix of zeros with eps 0: 0 / 0, as the definition says
    const double inv = 1.0 / (sqrt(trace) + (double)poly.eps);
    for (int e = tid; e < blocks * 64; e += THREADS) {
        const int i = (s_block[e >> 6] >> 8) * 8 + ((e & 63) >> 3), j = (s_block[e >> 6] & 255) * 8 + (e & 7);
        const double v = s_t[e] * inv * inv;
        if (i >= j) s_a[i * pitch + j] = s_a[j * pitch + i] = v;
    }
    __syncthreads();

    for (int s = 0; s < poly.steps; ++s) {
        const bool last = s + 1 == poly.steps;
        for (int t = warp; t < blocks; t += WARPS) small_product<true>(s_a, s_a, s_q, np, pitch, s_block[t], lane, poly.c, poly.b, poly.a);  // Q
        __syncthreads();
        // unless it is the last step, A = (Q A) Q; P = Q P (P = Q in the first step)
        const int first = last ? blocks : 0, total = s == 0 ? blocks : 2 * blocks;
        for (int t = first + warp; t < total; t += WARPS) {
            if (t < blocks) small_product<false>(s_q, s_a, s_t, np, pitch, s_block[t], lane, 0.0, 0.0, 0.0);
            else small_product<false>(s_q, s_p, s_own, np, pitch, s_block[t - blocks], lane, 0.0, 0.0, 0.0);
        }
        if (s == 0)
            for (int e = tid; e < size; e += THREADS) s_p[e] = s_q[e];
        __syncthreads();
        if (s > 0) {
            double* z = s_p;
            s_p = s_own;
            s_own = z;
        }
        if (!last) {
            for (int t = warp; t < blocks; t += WARPS) small_product<false>(s_t, s_q, s_a, np, pitch, s_block[t], lane, 0.0, 0.0, 0.0);
            __syncthreads();
        }
    }

    // out = P U / (|U| + eps), 8 rows x 8 columns per warp
    for (int64_t j0 = begin; j0 < end; j0 += jc_max) {
        const int jc = (int)min((int64_t)jc_max, end - j0), jp = (jc + 7) / 8 * 8;
        if (end - begin > jc_max) {  // else they are still there
            __syncthreads();
            small_fill<T, false, THREADS>(io, b, n, np, tall, j0, jc, jp, s_x, pitch);
            __syncthreads();
        }
        for (int t = warp; t < side * (jp / 8); t += WARPS) {
            const int bi = t % side, bj = t / side, i = bi * 8 + (lane >> 2), j = bj * 8 + 2 * (lane & 3);
            const int64_t at = b * io.out_batch + (tall ? (j0 + j) * io.out_stride + i : i * io.out_stride + j0 + j), next = tall ? io.out_stride : 1;
            float w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) w[q] = io.m && i < n && j + q < jc ? io.w[at + q * next] : 0.0f;
            const double *p = s_p + (lane & 3) * pitch + bi * 8 + (lane >> 2), *x = s_x + (bj * 8 + (lane >> 2)) * pitch + (lane & 3);
            double c[2][2] = {{0.0, 0.0}, {0.0, 0.0}};
#pragma unroll 4
            for (int k = 0; k < np; k += 8) {
                small_mma(c[0], p[k * pitch], x[k]);
                small_mma(c[1], p[(k + 4) * pitch], x[k + 4]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
                if (i < n && j + q < jc) orth_store<T>(io, at + q * next, w[q], (float)((c[0][q] + c[1][q]) * inv));
        }
    }
}

// How many clusters of sixteen (which are not portable) the current device runs at once at the largest shared memory: asked once per device.
template <typename T, int WARPS>
int small_clusters() {
    static std::atomic<int> known[64];  // 0 not asked, else one more
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int k = known[dev].load();
    if (!k) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(SMALL_CLUSTER);
        cfg.blockDim = dim3(32 * WARPS);
        cfg.dynamicSmemBytes = SMALL_SMEM;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = SMALL_CLUSTER;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int fit = 0;
        const bool ok = cudaFuncSetAttribute(k_orth_small<T, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM) == cudaSuccess &&
                        cudaFuncSetAttribute(k_orth_small<T, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&fit, k_orth_small<T, WARPS>, &cfg) == cudaSuccess && fit >= 1;
        if (!ok) cudaGetLastError();
        known[dev].store(k = (ok ? fit : 0) + 1);
    }
    return k - 1;
}

// CTAs per matrix: 32 columns or more for each, and no more than the chip holds at once (sixteen for eight: n = 32, m = 1024 in 16 us for 20); most: of a cluster
int small_ctas(const OrthIo& io, int64_t m, int most) {
    int cs = 1;
    while (cs < most && cs * 32 < m && (int64_t)io.batch * 2 * cs <= sm_count()) cs *= 2;
    return cs;
}
template <typename T, int WARPS>
void small_launch(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int n, int64_t m, int cs) {
    // a CTA's columns stay in shared memory where they fit beside the matrices; the partial sums take 64 doubles per warp of the matrices
    const int np = (n + 7) / 8 * 8, pitch = small_pitch(np), three = np * pitch * 3, part = 64 * WARPS;
    const int matrices = np * pitch * 2 + (three > part ? three : part), room = (SMALL_SMEM / 8 - matrices) / pitch / 8 * 8;
    const int64_t per = (m + cs - 1) / cs;
    const int jc_max = per < room ? (int)((per + 7) / 8 * 8) : room;
    const size_t smem = (size_t)(jc_max * pitch + matrices) * sizeof(double);
    if (!small_clusters<T, WARPS>()) op_note(cudaFuncSetAttribute(k_orth_small<T, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM));  // else it is set
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cs, (unsigned)io.batch);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    op_note(cudaLaunchKernelEx(&cfg, k_orth_small<T, WARPS>, io, p, jc_max));
}
// Sixteen warps where the products or the loads keep them busy (64 x 512: 44 us, with ten 50, eight 47; 15 of 19 x 2200: 18, 20, 21; 9 of 24 x 1536: 16.0, with eight 17.5), else eight, whose columns
// are one batch of loads: fewer to wait for at a barrier (16 x 64: 9.1 us, 10.1), and two CTAs per SM (9 of 16 x 1536: 12.5 us, with sixteen 21.6: the ninth cluster has to wait).
template <typename T>
void orth_small_go(cudaStream_t s, const OrthIo& io, const OrthPoly& p) {
    const int n = io.rows < io.cols ? io.rows : io.cols;
    const int64_t m = io.rows < io.cols ? io.cols : io.rows;
    const int few = small_ctas(io, m, small_clusters<T, 8>() > 0 ? SMALL_CLUSTER : 8);
    if (n <= 24 && (n + 7) / 8 * 8 * ((m + few - 1) / few) <= 256 * SMALL_BATCH) return small_launch<T, 8>(s, io, p, n, m, few);
    small_launch<T, 16>(s, io, p, n, m, small_ctas(io, m, io.batch <= small_clusters<T, 16>() ? SMALL_CLUSTER : 8));
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

// More elements than any device holds are refused, before the sizes of what is derived from them could wrap.
#define ORTH_MAX_ELEMENTS (1LL << 40)
bool orth_sizes(int batch, int rows, int cols) {
    return batch >= 0 && batch <= 65535 && rows >= 1 && cols >= 1 && (int64_t)rows * cols <= ORTH_MAX_ELEMENTS / (batch > 0 ? batch : 1);
}

int orth_check(int type, int batch, int rows, int cols, const OrthPoly& p, char* err, size_t err_len) {
    if (!op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (!orth_sizes(batch, rows, cols))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "batch must be in [0, 65535], rows and cols positive, and batch * rows * cols at most 2^40");
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
    if (type == TB_TYPE_F32) orth_small_go<float>(s, io, p);
    else if (type == TB_TYPE_F16) orth_small_go<__half>(s, io, p);
    else orth_small_go<__nv_bfloat16>(s, io, p);
}

extern "C" int64_t tb_orthogonalise_workspace(int type, int batch, int rows, int cols) {
    if (!op_type_size(type) || !orth_sizes(batch, rows, cols)) return TB_ERR_INVALID_ARGUMENT;
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
    if (!op_apart(d_x, x_batch, x_stride, d_out, out_batch, out_stride, batch, rows, cols, op_type_size(type))) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_out overlaps d_x in part");
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
    if (!orth_sizes(batch, rows, cols)) return TB_ERR_INVALID_ARGUMENT;
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
    // a result may be its input's memory and must not touch any other tensor's
    const uintptr_t count = (uintptr_t)batch * rows * cols;
    const auto apart = [](const void* a, uintptr_t a_bytes, const void* b, uintptr_t b_bytes) { return (uintptr_t)a + a_bytes <= (uintptr_t)b || (uintptr_t)b + b_bytes <= (uintptr_t)a; };
    const uintptr_t f = count * 4, gb = count * op_type_size(g_type);
    if ((d_w_out != d_w && !apart(d_w_out, f, d_w, f)) || (d_m_out != d_m && !apart(d_m_out, f, d_m, f)) || !apart(d_w_out, f, d_m_out, f) || !apart(d_w_out, f, d_m, f) ||
        !apart(d_m_out, f, d_w, f) || !apart(d_g, gb, d_w_out, f) || !apart(d_g, gb, d_m_out, f))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
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
