// The forward pass of the root-mean-square norm (rms_kernels.cu has the mathematics): the kernels of both outputs, which are compiled apart, in the tensors' type by
// rms_kernels.cu and in 8 bits by rms_quantised.cu.
#pragma once
#include "norm.cuh"

#include <cuda_fp8.h>

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
void rms_quantised_run(const RmsForward& a, int type, bool wide);  // rms_quantised.cu

namespace {

// The longest row that the backward pass keeps in registers (the forward pass: 32768, the last of rms_forward_pick).  Kept and read again: forward 2000 x 17000 fp32 56 and 63 us, 24576 bf16 48 and 67; backward 2000 x
// 16384 fp32 105 and 119, but 2000 x 10000 86 and 82, 200 x 12288 26 and 22.
#define RMS_REG_N_BACK 16384
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
// Its inverse, NaN of a scale that is infinite (0 would make the group's other numbers zeros)
__device__ __forceinline__ float rms_inverse(float s) { return s < INFINITY ? 1.0f / s : __int_as_float(0x7fc00000); }
// Whether z of largest magnitude `most` may be multiplied with 448 / most for z late / s: to 2 ulp, where nothing leaves the range of that quotient and s is not the smallest scale.
// (With divisions to the last bit for every group, 40000 x 1000 fp16 in groups of 128 took 40 us.)
__device__ __forceinline__ bool rms_usual(float most, float late) { return most > 1e-30f && most < 1e30f && most * late > 1e-35f; }
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


// W warps per row, VEC adjacent columns per access, CH accesses per thread: a thread holds columns (c * LANES + t) * VEC + i.  With W = 1 a row has L lanes.
// G: 0 for y of type T, 1 for 8 bits with a scale per row, else columns that share a scale (with W = 1, or as many adjacent lanes of a warp).  FULL: accesses that are inside the row for every thread.  AHEAD: warps that walk down the rows, the next one's x on its way while they compute
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
            // z = f h * weight, y = z * late.  h * weight may leave fp32's range, or lose bits, where y does not, so 1 / rms comes first; in the kernels that walk down it may come last, at
            // one multiplication less per column, where z is no larger than y and less than 16 times smaller (40000 x 1000 fp16 in groups of 128: 24.7 us, 25.4 where it comes first).
            const bool near = AHEAD && r >= 1.0f && r < 16.0f;
            const float late = near ? r : 1.0f;
            if (!near)
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (c < FULL || (c * LANES + t) * VEC < n) rms_multiply<VEC>(v[c], r);
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
            constexpr int GL = G > 1 ? (G / VEC < L ? G / VEC : L) : L, JOIN = G > 1 ? G / (GL * VEC) : 1;  // lanes and accesses that share a scale
            static_assert(JOIN == 1 || W == 1, "the next access is other columns of the group in the same lanes");
            const int groups = G > 1 ? (n + G - 1) / G : 1;
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
                usual = rms_usual(most[0], late);
                if (t == 0 && there) scale_out[row] = rms_scale(most[0] * late);
            } else {
#pragma unroll
                for (int c = 0; c < CH; c += JOIN) {
                    const int col = (c * LANES + t) * VEC;
#pragma unroll
                    for (int k = 1; k < JOIN; ++k)
                        if (c + k < CH) most[c] = rms_larger(most[c], most[c + k < CH ? c + k : 0]);
                    most[c] = rms_group_max<GL>(most[c]);
#pragma unroll
                    for (int k = 1; k < JOIN; ++k)
                        if (c + k < CH) most[c + k < CH ? c + k : 0] = most[c];
                    usual = usual && (rms_usual(most[c], late) || (c >= FULL && col >= n));
                    if (there && (c < FULL || col < n) && t % GL == 0) scale_out[row * groups + col / G] = rms_scale(most[c] * late);
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
                    rms_multiply<VEC>(v[k], late);
                    rms_store_q<VEC>(q + col, v[k], rms_inverse(rms_scale(most[G == 1 ? 0 : k] * late)));
                }
            }
        }
    } while (AHEAD && (row += (int64_t)gridDim.x * RB) < rows);
}

// Any row: a block per row that reads it again for every pass; thread t takes columns t, t + TH, ..  Rows longer than 32768, and 8-bit rows over 1536 columns that start anywhere.
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
        const float s = rms_scale(most), inverse = rms_inverse(s);
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
        const float s = rms_scale(rms_group_max<32>(most)), inverse = rms_inverse(s);
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
    // Few rows: as many warps for each as leave a thread eight columns or sixteen (47 x 1189 fp16 rows that start anywhere: 8.5 us with a warp per row)
    if constexpr (G <= 1)
        if (a.n > 512 && a.rows <= 2 * (int64_t)sm_count()) {
            GO(512, 4, 32, 8); GO(1024, 8, 32, 8); GO(2048, 16, 32, 8); GO(4096, 32, 32, 8); GO(8192, 32, 32, 16);
        }
    if constexpr (G <= 32) GO(0, 1, 8, 8);  // a group is shorter than the row
    if constexpr (G <= 64) GO(0, 1, 16, 8);
    GO(0, 1, 32, 8); GO(256, 1, 32, 16);
    if constexpr (VEC > 1) { GO(512, 1, 32, 24); GO(768, 1, 32, 32); }
    else GO(512, 1, 32, 32);
    // many rows of 16-byte accesses (65536 x 1088 bf16 48 us, four warps per row 70; 1536 fp32 119 and 116); not the best for some hundreds of rows (500 x 1536 fp32 4.4 and 2.5), nor for single elements (30000 x 1251 bf16 65
    // and 48)
    GO(1024, 1, 32, 48);
    if constexpr (VEC > 1 || G <= 1) {
        if constexpr (G == 0) { GO(1536, 4, 32, 16); GO(2048, 4, 32, 32); }
        else GO(1536, 4, 32, 32);
        GO(4096, 8, 32, 32); GO(8192, 16, 32, 32); GO(16384, 32, 32, 32);
    }
#undef GO
    rms_forward_any<T>(a);
}

}  // namespace
