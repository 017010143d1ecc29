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
#include "norm.cuh"

#include <cuda_fp8.h>

namespace {

#define RMS_REG_N 32768      // longest row that the forward pass keeps in registers
#define RMS_REG_N_BACK 16384 // ... the backward pass
#define RMS_MOST 448.0f      // the largest e4m3 number
#define RMS_LEAST 1.17549435e-38f  // 2^-126: the smallest scale

// 1 / sqrt(mean of squares + eps) by `sum(f)`, the row's sum of (f h)^2 over its threads, the same in all of them; `any(c)`: whether c holds in a row that
// shares the sums' barriers or shuffles.  Squares overflow above 2^63 and lose bits below 2^-75, which counts where eps is no larger.  `scale` is the f
// that was taken, and what comes back is 1 / rms of f h: the row's own is f times that.
template <typename Sum, typename Any>
__device__ __forceinline__ float rms_factor(int n, float eps, float& scale, Sum sum, Any any) {
    float ss = sum(1.0f), f = 1.0f;
    const bool large = ss > 8.5e37f, small = ss < 8e-25f && eps < 8e-31f;
    if (any(large || small)) {
        f = large ? 7.888609052e-31f : small ? 1.2676506002e30f : 1.0f;  // 2^-100, 2^100
        ss = sum(f);
    }
    scale = f;
    return 1.0f / sqrtf(ss / (float)n + eps * f * f);
}

// two fp32 operations at once
__device__ __forceinline__ uint64_t rms_pair(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
template <int N>
__device__ __forceinline__ void rms_multiply(float (&v)[N], const float (&w)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(rms_pair(v[i], v[i + 1])), "l"(rms_pair(w[i], w[i + 1])));
            v[i] = __uint_as_float((unsigned)r), v[i + 1] = __uint_as_float((unsigned)(r >> 32));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= w[i];
    }
}
template <int N>
__device__ __forceinline__ void rms_multiply(float (&v)[N], float by) {
    float w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = by;
    rms_multiply<N>(v, w);
}
// the sum of squares of a thread's columns: two chains, the even and the odd ones
template <int CH, int N>
__device__ __forceinline__ float rms_squares(const float (&v)[CH][N]) {
    if constexpr (N % 2 == 0) {
        uint64_t sum = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const uint64_t p = rms_pair(v[c][i], v[c][i + 1]);
                asm("fma.rn.f32x2 %0, %1, %1, %0;" : "+l"(sum) : "l"(p));
            }
        return __uint_as_float((unsigned)sum) + __uint_as_float((unsigned)(sum >> 32));
    } else {
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) sum = fmaf(v[c][i], v[c][i], sum);
        return sum;
    }
}
// the largest magnitude; NaN if any is
__device__ __forceinline__ float rms_larger(float a, float b, float c = 0.0f) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void rms_unpack(const OpRaw<T, N>& raw, float (&to)[N]) {
    if constexpr (std::is_same<T, __half>::value && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&raw.w[i / 2]));
            to[i] = two.x, to[i + 1] = two.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = raw.get(i);
    }
}
// the scale of a group from its largest |y|; NaN stays NaN
__device__ __forceinline__ float rms_scale(float most) {
    const float s = most * (1.0f / RMS_MOST);
    return s < RMS_LEAST ? RMS_LEAST : s;
}
// Whether z of largest magnitude `most` may be multiplied with 448 / most for z r / s: to 2 ulp, where nothing leaves the range of that quotient and s is not the smallest scale.
// (With divisions to the last bit for every group, 40000 x 1000 fp16 in groups of 128 took 40 us.)
__device__ __forceinline__ bool rms_usual(float most, float r) { return most > 1e-30f && most < 1e30f && most * r > 1e-35f; }
__device__ __forceinline__ uint8_t rms_q(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
// VEC numbers times `by` as adjacent bytes
template <int VEC>
__device__ __forceinline__ void rms_store_q(uint8_t* to, float (&v)[VEC], float by) {
    rms_multiply<VEC>(v, by);
    if constexpr (VEC == 1) {
        *to = rms_q(v[0]);
    } else {
        OpVec<unsigned, VEC / 4> u;
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const unsigned low = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
            const unsigned high = __nv_cvt_float2_to_fp8x2(make_float2(v[i + 2], v[i + 3]), __NV_SATFINITE, __NV_E4M3);
            u.v[i / 4] = low | high << 16;
        }
        *reinterpret_cast<OpVec<unsigned, VEC / 4>*>(to) = u;
    }
}

// the largest of G lanes' magnitudes, whose bits are ordered like them with NaN above all
template <int G>
__device__ __forceinline__ float rms_group_max(float most) {
    unsigned v = __float_as_uint(most);
    if constexpr (G == 32) return __uint_as_float(__reduce_max_sync(0xffffffffu, v));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __uint_as_float(v);
}

// VEC columns of the weight in one access: 32 bytes of eight columns, as adjacent as the lanes are.  (Two of 16 bytes with gaps of 16 between the lanes cost four times the
// wavefronts of the L1, more than all the rest of an 8-bit row: 40000 x 1000 fp16 37 us.)
template <int VEC>
__device__ __forceinline__ void rms_columns(const float* p, int col, float (&to)[VEC]) {
    if constexpr (VEC == 8) {
        if (p) {
            asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=f"(to[0]), "=f"(to[1]), "=f"(to[2]), "=f"(to[3]), "=f"(to[4]), "=f"(to[5]), "=f"(to[6]), "=f"(to[7])
                : "l"(p + col));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) to[i] = 1.0f;
        }
    } else {
        norm_columns<VEC>(p, col, 1.0f, to);
    }
}

struct RmsForward {
    cudaStream_t s;
    const void* x;
    int64_t xs;
    const void* r;  // NULL: none
    int64_t rs;
    const float* w;
    float eps;
    int64_t rows;
    int n;
    void* y;        // or the 8-bit numbers
    int64_t ys;
    void* h;        // NULL: not wanted
    int64_t hs;
    float* rstd;
    float* scale;   // of 8-bit numbers: [rows][groups]
    int group;      // 0: y is of the tensors' type
};

// W warps per row, VEC adjacent columns per access, CH accesses per thread: a thread holds columns (c * LANES + t) * VEC + i.  With W = 1 a row has L lanes.
// G: 0 for y of type T, 1 for 8 bits with a scale per row, else lanes that share a scale.  FULL: accesses that are inside the row for every thread.  AHEAD: warps that walk down the rows, the next one's x on its way while they compute
// (16-bit rows without a residual, where instructions take as long as the bytes); otherwise every group of lanes has one row.
constexpr int rms_per_sm(int columns) { return columns <= 32 ? 7 : 5; }  // of blocks that walk down, by a thread's columns

template <typename T, int W, int L, int VEC, int CH, int FULL, int G, bool AHEAD>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32, AHEAD ? rms_per_sm(CH * VEC) : 1)
k_rms_forward(const T* x, int64_t x_stride, const T* res, int64_t res_stride, const float* weight, float eps, int64_t rows, int n, void* y, int64_t y_stride,
              T* h, int64_t h_stride, float* __restrict__ rstd_out, float* __restrict__ scale_out) {
    constexpr int LANES = W == 1 ? L : 32 * W, SUBS = W == 1 ? 32 / L : 1, RB = W == 1 ? 4 * SUBS : 1;  // rows per block
    __shared__ float s_sum[2][W];
    __shared__ float s_max[W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = W == 1 ? lane % L : threadIdx.x;
    int64_t row = (int64_t)blockIdx.x * RB + (W == 1 ? warp * SUBS + lane / L : 0);
    op_next_may_start();
    if (L == 32 && row >= rows) return;  // by whole warps; lanes that share a warp stay for its sums
    const bool there = L == 32 || row < rows;
    OpRaw<T, VEC> xv[CH], rv[CH];
    const auto load = [&](OpRaw<T, VEC>(&to)[CH], const T* from) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LANES + t) * VEC;
            to[c].zero();
            if (there && (c < FULL || col < n)) to[c].load(from + col);
        }
    };
    op_wait_for_previous();
    load(xv, x + row * x_stride);
    do {
        if (!AHEAD && res) load(rv, res + row * res_stride);
        float v[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            rms_unpack(xv[c], v[c]);
            if (!AHEAD && res) {
                float u[VEC];
                rms_unpack(rv[c], u);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[c][i] += u[i];
            }
        }
        if (AHEAD && row + (int64_t)gridDim.x * RB < rows) load(xv, x + (row + (int64_t)gridDim.x * RB) * x_stride);
        if (!AHEAD && h && there) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LANES + t) * VEC;
                if (c < FULL || col < n) op_store<T, VEC>(h + row * h_stride + col, v[c]);
            }
        }
        int turn = 0;
        float f;
        const float r = rms_factor(
            n, eps, f,
            [&](float by) {
                float ss[1];
                if (turn) {  // the second sum: f h stays
#pragma unroll
                    for (int c = 0; c < CH; ++c) rms_multiply<VEC>(v[c], by);
                }
                ss[0] = rms_squares(v);
                norm_rows_sum<W, L, 1>(ss, s_sum[turn++ & 1], warp, lane);
                return ss[0];
            },
            [](bool c) { return W == 1 && L < 32 ? __any_sync(0xffffffffu, c) : c; });
        if (t == 0 && there && rstd_out) rstd_out[row] = f * r;
        if constexpr (G == 0) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LANES + t) * VEC;
                if (c >= FULL && col >= n) continue;
                rms_multiply<VEC>(v[c], r);
                if (weight) {
                    float w[VEC];
                    rms_columns<VEC>(weight, col, w);
                    rms_multiply<VEC>(v[c], w);
                }
                if (there) op_store<T, VEC>(static_cast<T*>(y) + row * y_stride + col, v[c]);
            }
        } else {
            // z = f h * weight, y = z * r: one multiplication less for every column
            if (weight) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LANES + t) * VEC;
                    if (c >= FULL && col >= n) continue;
                    float w[VEC];
                    rms_columns<VEC>(weight, col, w);
                    rms_multiply<VEC>(v[c], w);
                }
            }
            float most[CH];  // columns that do not exist are zeros
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                most[c] = 0.0f;
#pragma unroll
                for (int i = 0; i < VEC; i += 2) most[c] = rms_larger(most[c], v[c][i], VEC > 1 ? v[c][(i + 1) % VEC] : 0.0f);
            }
            uint8_t* q = static_cast<uint8_t*>(y) + row * y_stride;
            const int groups = G > 1 ? (n + G * VEC - 1) / (G * VEC) : 1;
            bool usual = true;
            if constexpr (G == 1) {
#pragma unroll
                for (int c = 1; c < CH; ++c) most[0] = rms_larger(most[0], most[c]);
                most[0] = rms_group_max<L>(most[0]);
                if (W > 1) {
                    if (lane == 0) s_max[warp] = most[0];
                    __syncthreads();
#pragma unroll
                    for (int w = 0; w < W; ++w) most[0] = rms_larger(most[0], s_max[w]);
                }
                usual = rms_usual(most[0], r);
                if (t == 0 && there) scale_out[row] = rms_scale(most[0] * r);
            } else {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LANES + t) * VEC;
                    most[c] = rms_group_max<G>(most[c]);
                    usual = usual && (rms_usual(most[c], r) || (c >= FULL && col >= n));
                    if (there && (c < FULL || col < n) && t % G == 0) scale_out[row * groups + col / (G * VEC)] = rms_scale(most[c] * r);
                }
            }
            if (__all_sync(0xffffffffu, usual || !there)) {
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LANES + t) * VEC;
                    if (there && (c < FULL || col < n)) rms_store_q<VEC>(q + col, v[c], __fdividef(RMS_MOST, most[G == 1 ? 0 : c]));
                }
                continue;
            }
#pragma unroll 1
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LANES + t) * VEC;
#pragma unroll
                for (int k = 0; k < CH; ++k) {
                    if (k != c || !there || col >= n) continue;
                    rms_multiply<VEC>(v[k], r);
                    rms_store_q<VEC>(q + col, v[k], 1.0f / rms_scale(most[G == 1 ? 0 : k] * r));
                }
            }
        }
    } while (AHEAD && (row += (int64_t)gridDim.x * RB) < rows);
}

// Any row: a block per row that reads it again for every pass; thread t takes columns t, t + TH, ..  Rows longer than RMS_REG_N, and 8-bit rows that start anywhere.
// C counts columns: int, or int64_t where the last step would go beyond 2^31.
template <typename T, typename C, int TH>
__global__ void __launch_bounds__(TH)
k_rms_forward_long(const T* x, int64_t x_stride, const T* res, int64_t res_stride, const float* weight, float eps, int n, void* y, int64_t y_stride, T* h, int64_t h_stride,
                   float* __restrict__ rstd_out, float* __restrict__ scale_out, int group) {
    constexpr int W = TH / 32;
    __shared__ float s_sum[2][W];
    __shared__ float s_max[W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *rr = res + row * res_stride;
    T* hr = h + row * h_stride;
    op_next_may_start();
    op_wait_for_previous();
    const auto sum_at = [&](C c) { return res ? op_float(xr[c]) + op_float(rr[c]) : op_float(xr[c]); };
    int turn = 0;
    float f;
    const float r = rms_factor(
        n, eps, f,
        [&](float by) {
            float ss = 0.0f;
            for (C c = threadIdx.x; c < n; c += TH) {
                const float v = sum_at(c) * by;
                ss = fmaf(v, v, ss);
            }
            return norm_row_sum<W>(ss, s_sum[turn++ & 1], warp, lane);
        },
        [](bool c) { return c; });
    if (threadIdx.x == 0 && rstd_out) rstd_out[row] = f * r;
    const auto y_at = [&](C c, float v) { return v * f * r * (weight ? weight[c] : 1.0f); };
    if (group == 0) {
        T* yr = static_cast<T*>(y) + row * y_stride;
        for (C c = threadIdx.x; c < n; c += TH) {
            const float v = sum_at(c);
            if (h) hr[c] = op_round<T>(v);
            yr[c] = op_round<T>(y_at(c, v));
        }
        return;
    }
    uint8_t* q = static_cast<uint8_t*>(y) + row * y_stride;
    if (group >= n) {
        float most = 0.0f;
        for (C c = threadIdx.x; c < n; c += TH) most = rms_larger(most, y_at(c, sum_at(c)));
        most = rms_group_max<32>(most);
        if (lane == 0) s_max[warp] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) most = rms_larger(most, s_max[w]);
        const float s = rms_scale(most), inverse = 1.0f / s;
        if (threadIdx.x == 0) scale_out[row] = s;
        for (C c = threadIdx.x; c < n; c += TH) {
            const float v = sum_at(c);
            if (h) hr[c] = op_round<T>(v);
            q[c] = rms_q(y_at(c, v) * inverse);
        }
        return;
    }
    // a warp per group of up to 128 columns
    const int groups = (int)(((C)n + group - 1) / group);
    for (int g = warp; g < groups; g += W) {
        float v[4];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const C c = (C)g * group + i * 32 + lane;
            v[i] = 0.0f;
            if (i * 32 < group && c < n) {
                const float u = sum_at(c);
                if (h) hr[c] = op_round<T>(u);
                v[i] = y_at(c, u);
            }
            most = rms_larger(most, v[i]);
        }
        const float s = rms_scale(rms_group_max<32>(most)), inverse = 1.0f / s;
        if (lane == 0) scale_out[row * groups + g] = s;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const C c = (C)g * group + i * 32 + lane;
            if (i * 32 < group && c < n) q[c] = rms_q(v[i] * inverse);
        }
    }
}

template <typename T, int W, int L, int VEC, int CH, int FULL, int G>
void rms_forward_go(const RmsForward& a) {
    const int64_t per = W == 1 ? 128 / L : 1, blocks = (a.rows + per - 1) / per, most = (int64_t)sm_count() * rms_per_sm(CH * VEC);
#define RUN(AHEAD, BLOCKS)                                                                                                                                              \
    op_launch_next(a.s, dim3((unsigned)(BLOCKS)), dim3(W == 1 ? 128 : W * 32), 0, k_rms_forward<T, W, L, VEC, CH, FULL, G, AHEAD>, (const T*)a.x, a.xs, (const T*)a.r, a.rs, a.w, a.eps, a.rows, a.n, a.y, \
                   a.ys, (T*)a.h, a.hs, a.rstd, a.scale)
    if constexpr (sizeof(T) == 2 && W == 1 && L == 32 && VEC > 1)
        if (!a.r && blocks > most) return RUN(true, most);
    RUN(false, blocks);
#undef RUN
}
template <typename T>
void rms_forward_any(const RmsForward& a) {
    const bool counts = a.n <= INT32_MAX - 1023;
#define ANY(TH) \
    op_launch_next(a.s, dim3((unsigned)a.rows), dim3(TH), 0, counts ? k_rms_forward_long<T, int, TH> : k_rms_forward_long<T, int64_t, TH>, (const T*)a.x, a.xs, (const T*)a.r, a.rs, a.w, a.eps, a.n, a.y, a.ys, \
                   (T*)a.h, a.hs, a.rstd, a.scale, a.group)
    if (a.n <= 2048) ANY(128);
    else ANY(1024);
#undef ANY
}
template <typename T, int VEC, int G>
void rms_forward_pick(const RmsForward& a) {
    // the rows over LO columns, up to W * K * L
#define GO(LO, W, L, K) \
    if (a.n <= (W) * (K) * (L)) return rms_forward_go<T, W, L, VEC, ((K) + VEC - 1) / VEC, (LO) / ((W) * (L) * VEC), G>(a)
    if constexpr (G <= 1 || G * VEC <= 32) GO(0, 1, 8, 8);  // a group is shorter than the row
    if constexpr (G <= 1 || G * VEC <= 64) GO(0, 1, 16, 8);
    GO(0, 1, 32, 8); GO(256, 1, 32, 16); GO(512, 1, 32, 24); GO(768, 1, 32, 32); GO(1024, 1, 32, 48);
    GO(1536, 4, 32, 16); GO(2048, 4, 32, 32); GO(4096, 8, 32, 32); GO(8192, 16, 32, 32); GO(16384, 32, 32, 32);
#undef GO
    rms_forward_any<T>(a);
}
template <typename T, int VEC>
void rms_forward_type(const RmsForward& a, bool wide) {
    if (a.group == 0) return wide ? rms_forward_pick<T, VEC, 0>(a) : rms_forward_pick<T, 1, 0>(a);
    if (!wide) return rms_forward_any<T>(a);
    if (a.group >= a.n) return rms_forward_pick<T, VEC, 1>(a);
    if (a.group == 32) rms_forward_pick<T, VEC, 32 / VEC>(a);
    else if (a.group == 64) rms_forward_pick<T, VEC, 64 / VEC>(a);
    else rms_forward_pick<T, VEC, 128 / VEC>(a);
}

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
// Blocks: at most what runs at once; 16 rows or more for each, or the blocks' rows of gradients cost as much as the rows themselves, but one per SM as far as the rows go.
int rms_backward_blocks(int64_t rows, int n) {
    if (n > RMS_REG_N_BACK) return (int)(rows < 64 ? (rows < 1 ? 1 : rows) : 64);
    const int w = rms_warps_back(n);
    const int64_t turn = n <= 64 ? 32 : n <= 128 ? 16 : w == 1 ? 8 : n <= 4096 ? 2 : 1, sms = sm_count(), most = sms * rms_per_sm_back(w);
    const int64_t turns = (rows + turn - 1) / turn, least = (16 + turn - 1) / turn, want = (turns + least - 1) / least;
    if (turns <= 2) return 1;  // no second launch then
    const int64_t few = turns < sms ? turns : sms;
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
    if (type == TB_TYPE_F32) rms_forward_type<float, 4>(a, wide);
    else if (type == TB_TYPE_F16) rms_forward_type<__half, 8>(a, wide);
    else rms_forward_type<__nv_bfloat16, 8>(a, wide);
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
