// Newton-Schulz steps of matrices with a short side above 64: products on the 5th-generation tensor cores.
//
// Operands are fp16 "limbs" of numbers scaled by 2^11: one limb holds 11 bits of a number, two hold 22 (the second is the first one's rounding error, times
// 2^11 once more, so that it leaves the range of fp16 no sooner than the first).  That is so from 2^-25 on, the matrix's norm being 1; below, one limb is off by at
// most 2^-36 and two by 2^-47.  With two limbs a product is three products of limbs (high low, low high, high high; low low is below 2^-22) into one
// fp32 accumulator, which the first high product scales back by 2^-11: the steps keep fp32 accuracy, for blocks and rows far below the norm too, at a third of
// the fp16 rate; fp32 on the CUDA cores has a thirtieth.  (The second limb at the first one's scale left the range sooner: a block of 1e-5 of another came
// out 2e-4 off, now 2e-7.)  With one limb the roundings (2^-12 of an element, a few times over: 1.0e-3 to 1.3e-3 of a result) stay below those of a bf16
// result (2^-9 of an element, 1.7e-3), at a third of the products: half of the time of two limbs at 4 x 1000 x 777, a third at 4096 x 4096.  Numbers up to 32
// fit; the entry points refuse coefficients that could leave that range.
//
// All matrices live in the workspace as 16 KB tiles of 128 rows x 64 columns, stored as the tensor cores want them in shared memory
// (rows of 128 bytes, their 16-byte pieces permuted by the row's last three bits), so every operand is fetched by untiled bulk copies
// and nothing is laid out twice:
//   Gram    A = X X^T             X's tiles as rows (K along the columns), both sides
//   square  Q = a I + b A + c A A A is symmetric: its rows serve as columns
//   apply   X = Q X               X's tiles as K x N operands (N along the columns): the same bytes, the other major
// Gram and square are symmetric: only tiles on and below the diagonal are computed, the epilogue stores the mirrored tile too.
// a I is part of Q, so that no product has to add its own input.
//
// One thread issues the bulk copies into a ring of stages, one the MMAs, eight warps read the accumulators from tensor memory.  The tensor
// cores truncate when they add to an accumulator: with two limbs that left 2.5e-5 of the result after five steps of K = 1000, 1.4e-5 with a new accumulator
// every 256 columns of K.  So it changes with every chunk of 64, which adds the small products first and the four large ones last, and the
// warps add what it held to their registers, rounded to nearest, while the next one fills.
// Every wait is bounded.  An accumulator is announced only when all of its MMAs were issued on operands that have arrived; a warp that waits in vain for one
// takes NaN for it, and stores those once the copies and MMAs that were under way are done: what a block stores is right or NaN.
//
// Measured, 4096 x 4096 in fp32: Gram 155 us, square 172, apply 290 (1.4 PFLOP/s of limb products, tensor pipe 76 to 92 % busy), last product with
// the weight update 331; the whole Muon step 3.7 to 3.85 ms, where the chip's power limit, not the kernel, sets the clock.  bf16: 1.25 ms.  Small
// products are bound by what surrounds the MMAs: 4 x 1000 x 777 bf16 takes 131 us in 17 launches of 7 to 9 us, 3 to 4 us of each inside the K loop.
#include "orth.cuh"

#include <atomic>

namespace {

#define OT_TILE 16384           // bytes of a tile of 128 x 64 fp16
#define OT_SCALE 2048.0f
#define OT_UNSCALE (1.0f / (2048.0f * 2048.0f))
#define OT_LOW_BITS 11          // of the second limb's further scale
#define OT_LOW ((float)(1 << OT_LOW_BITS))
#define OT_PARTS 8             // most parts of a Gram product
#define OT_NORM_BLOCKS 512      // most partial sums of squares per matrix
enum { OT_GRAM = 0, OT_SQUARE = 1, OT_APPLY = 2, OT_LAST = 3, OT_GRAM_PART = 4 };
// Who waits: the warp that copies, the one that issues the MMAs, the odd block's that tells it of its operands, those that read the accumulators; and any of
// them, in the end, for what is under way.
enum { OT_COPIES = 0, OT_PRODUCTS = 1, OT_RELAY = 2, OT_SUMS = 3, OT_END = 4 };
#ifndef OT_WAIT_LIMIT  // tries before a wait gives up; the last one outlasts the others
#define OT_WAIT_LIMIT(role) ((role) == OT_END ? 1 << 22 : 1 << 20)
#endif

__device__ __forceinline__ unsigned ot_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ot_bar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
template <int ROLE>
__device__ __forceinline__ bool ot_wait(unsigned bar, unsigned parity) {
    for (int i = 0; i < OT_WAIT_LIMIT(ROLE); ++i) {
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}
__device__ __forceinline__ void ot_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ot_copy(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Arrives at the same barrier of block `rank` of the cluster.  What it announces are operands that copies have brought (their bytes were counted
// before this thread arrives) or accumulators that have been read; no store of this thread's.  A release at cluster scope waits for the copies in
// flight as well: it made a chunk of 256 x 256 tiles of one limb take 1250 cycles instead of 500.
__device__ __forceinline__ void ot_arrive_at(unsigned bar, unsigned rank) {
    asm volatile(
        "{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %0, %1;\n\tmbarrier.arrive.shared::cluster.b64 _, [at];\n\t}" ::"r"(bar), "r"(rank)
        : "memory");
}
__device__ __forceinline__ void ot_cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// true in one lane of a whole warp, always the same one
__device__ __forceinline__ bool ot_elect() {
    unsigned one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// d = a b + d 2^-DOWN, or a b alone
template <int CTAS, int DOWN>
__device__ __forceinline__ void ot_mma(unsigned d, unsigned long long da, unsigned long long db, unsigned idesc, unsigned accumulate) {
    if (CTAS == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, %5;\n\t}" ::"r"(d), "l"(da), "l"(db),
                     "r"(idesc), "r"(accumulate), "n"(DOWN)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, %5;\n\t}" ::"r"(d), "l"(da), "l"(db),
                     "r"(idesc), "r"(accumulate), "n"(DOWN)
                     : "memory");
}
// arrives at the barrier (of both blocks) when the MMAs issued so far are done
template <int CTAS>
__device__ __forceinline__ void ot_commit(unsigned bar) {
    if (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ot_read32(unsigned taddr, unsigned (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
        "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
          "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// shared-memory matrix descriptor: 128-byte swizzle (2 at bit 61), version 1 (bit 46), offsets in 16 bytes
__device__ __forceinline__ unsigned long long ot_desc(unsigned addr, unsigned lbo, unsigned sbo) {
    return (unsigned long long)((addr & 0x3FFFFu) >> 4) | ((unsigned long long)(lbo >> 4) << 16) | ((unsigned long long)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// limbs of x: hi + lo / OT_LOW = x to 22 bits
template <int LIMBS>
__device__ __forceinline__ void ot_split(float x, __half (&h)[LIMBS]) {
    h[0] = __float2half_rn(x);
    if (LIMBS == 2) h[LIMBS - 1] = __float2half_rn((x - __half2float(h[0])) * OT_LOW);
}
// ... of two neighbours, as they lie in a tile
template <int LIMBS>
__device__ __forceinline__ void ot_split(float x, float y, __half2 (&h)[LIMBS]) {
    h[0] = __floats2half2_rn(x, y);
    if (LIMBS == 2) {
        const float2 high = __half22float2(h[0]);
        h[LIMBS - 1] = __floats2half2_rn((x - high.x) * OT_LOW, (y - high.y) * OT_LOW);
    }
}
// byte offset of element (row, col) in a 128 x 64 tile
__device__ __forceinline__ int ot_at(int row, int col) { return row * 128 + ((((col >> 3) ^ row) & 7) << 4) + (col & 7) * 2; }

// ---- the norm and the tiles of the first X ----------------------------------------------------------------------------
// N adjacent elements of u, with MUON the momentum's update included in the FIRST pass; the loads of the gradient and of the momentum are separate from
// what follows them so that a caller can issue several (a branch on the momentum in front of every load kept them apart and made a third of the instructions)
template <typename T, int N, bool MUON>
struct OtPiece {
    OpRaw<T, N> g;
    float m[MUON ? N : 1];
    __device__ __forceinline__ void load(const T* from, const float* momentum) {
        g.load(from);
        if constexpr (MUON) {
            constexpr int STEP = N < 4 ? N : 4;
#pragma unroll
            for (int i = 0; i < N; i += STEP) {
                float t[STEP];
                op_load<float, STEP>(momentum + i, t);
#pragma unroll
                for (int k = 0; k < STEP; ++k) m[i + k] = t[k];
            }
        }
    }
    template <bool FIRST>
    __device__ __forceinline__ void finish(const OrthIo& io, float (&u)[N], float* momentum = nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = g.get(i);
        if constexpr (MUON) {
            if (FIRST) {
#pragma unroll
                for (int i = 0; i < N; ++i) m[i] = fmaf(io.beta, m[i], u[i]);
                constexpr int STEP = N < 4 ? N : 4;
#pragma unroll
                for (int i = 0; i < N; i += STEP) {
                    float t[STEP];
#pragma unroll
                    for (int k = 0; k < STEP; ++k) t[k] = m[i + k];
                    op_store<float, STEP>(momentum + i, t);
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = io.nesterov ? fmaf(io.beta, m[i], u[i]) : m[i];
        }
    }
};

// Sum of squares (64 bits) of a matrix cut into segments of `len` elements (a row, or 4096 of a matrix without gaps), dealt to the blocks; every
// thread has 16 elements on their way.  64 blocks with one element each took 270 us for 4096 x 4096, 8 times this.
template <typename T, int N, bool MUON>
__global__ void __launch_bounds__(256) k_orth_norm(OrthIo io, int64_t segments, int64_t len, int64_t total, double* __restrict__ partial) {
    __shared__ double s_sum[8];
    const int b = blockIdx.y;
    double sum = 0.0;
    op_next_may_start();
    op_wait_for_previous();
    for (int64_t seg = blockIdx.x; seg < segments; seg += gridDim.x) {
        const int64_t r = total ? 0 : seg, c0 = total ? seg * len : 0, end = total ? min(total, c0 + len) : len;
        const T* g = static_cast<const T*>(io.g) + b * io.g_batch + r * io.g_stride;
        const int64_t at = ((int64_t)b * io.rows + r) * io.cols;
        const float* m = MUON ? io.m + at : nullptr;
        for (int64_t c = c0 + threadIdx.x * N; c < end; c += 256 * 16) {
            OtPiece<T, N, MUON> piece[16 / N];
#pragma unroll
            for (int q = 0; q < 16 / N; ++q)
                if (c + q * 256 * N < end) piece[q].load(g + c + q * 256 * N, MUON ? m + c + q * 256 * N : nullptr);
#pragma unroll
            for (int q = 0; q < 16 / N; ++q)
                if (c + q * 256 * N < end) {
                    float u[N];
                    piece[q].template finish<true>(io, u, MUON ? io.m_out + at + c + q * 256 * N : nullptr);
#pragma unroll
                    for (int i = 0; i < N; ++i) sum = fma((double)u[i], (double)u[i], sum);
                }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += s_sum[w];
        partial[b * OT_NORM_BLOCKS + blockIdx.x] = sum;
    }
}

// One tile per block: X0 = u / (|u| + eps), n x m with n <= m, zeros beyond both.  A thread makes 16-byte pieces of the tile: of N adjacent elements each
// where rows of u are rows of X, of eight rows of u where they are columns (TALL), through shared memory then.
template <typename T, int LIMBS, int N, bool TALL, bool MUON>
__global__ void __launch_bounds__(256) k_orth_pack(OrthIo io, float eps, const double* __restrict__ partial, int n_partial, uint8_t* __restrict__ x, int64_t limb_bytes) {
    __shared__ __align__(128) uint8_t s_tile[TALL ? LIMBS : 1][TALL ? OT_TILE : 16];
    __shared__ double s_part[8];
    const int b = blockIdx.z;
    const int n = TALL ? io.cols : io.rows, m = TALL ? io.rows : io.cols;
    op_wait_for_previous();
    op_next_may_start();
    double v = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 256) v += partial[b * OT_NORM_BLOCKS + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    const int i0 = blockIdx.y * 128, j0 = blockIdx.x * 64;
    uint8_t* to = x + (int64_t)b * LIMBS * limb_bytes + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * OT_TILE;
    constexpr int P = 8 / N, PIECES = 4;  // accesses of a piece, pieces of a thread
    OtPiece<T, N, MUON> piece[PIECES][P];
    // piece k: rows 32 k below the first one's, or columns 16 k beside
    const int i = TALL ? threadIdx.x & 127 : threadIdx.x >> 3, j = TALL ? threadIdx.x >> 7 << 3 : (threadIdx.x & 7) << 3;
    const int64_t r = TALL ? j0 + j : i0 + i, c = TALL ? i0 + i : j0 + j;
    const T* g = static_cast<const T*>(io.g) + b * io.g_batch + r * io.g_stride + c;
    const float* mo = MUON ? io.m_out + ((int64_t)b * io.rows + r) * io.cols + c : nullptr;
    const int left = TALL ? (i0 + i < n ? m - j0 - j : 0) : m - j0 - j;  // columns of X from the first element on
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const bool in = TALL ? 16 * k + q < left : i0 + i + 32 * k < n && q * N < left;
            if (in) piece[k][q].load(g, mo);
            if (TALL) {  // one row of u after the other
                const int64_t step = q < 7 ? 1 : 9;
                g += step * io.g_stride;
                if (MUON) mo += step * io.cols;
            } else {
                const bool next = q == P - 1;
                g += next ? 32 * io.g_stride - (P - 1) * N : N;
                if (MUON) mo += next ? 32 * (int64_t)io.cols - (P - 1) * N : N;
            }
        }
    __syncthreads();
    v = s_part[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) v += s_part[w];
    // 2^11 / (|u| + eps), one more rounding of 2^-24; beyond fp32's range for norms near its ends, so in two factors, the first a power of two
    const double scale = (double)OT_SCALE / (sqrt(v) + (double)eps);
    const float inv0 = scale > 0x1p100 ? 0x1p64f : scale < 0x1p-100 ? 0x1p-64f : 1.0f, inv = (float)(scale / (double)inv0);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        float u[8];
#pragma unroll
        for (int q = 0; q < P; ++q) {
            float t[N];
#pragma unroll
            for (int e = 0; e < N; ++e) t[e] = 0.0f;
            if (TALL ? 16 * k + q < left : i0 + i + 32 * k < n && q * N < left) piece[k][q].template finish<false>(io, t);
#pragma unroll
            for (int e = 0; e < N; ++e) u[q * N + e] = t[e] * inv0 * inv;
        }
        unsigned out[LIMBS][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            __half2 h[LIMBS];
            ot_split<LIMBS>(u[2 * e], u[2 * e + 1], h);
#pragma unroll
            for (int l = 0; l < LIMBS; ++l) out[l][e] = *reinterpret_cast<const unsigned*>(&h[l]);
        }
#pragma unroll
        for (int l = 0; l < LIMBS; ++l)
            *reinterpret_cast<uint4*>((TALL ? &s_tile[l][0] : to + l * limb_bytes) + ot_at(TALL ? i : i + 32 * k, TALL ? j + 16 * k : j)) =
                make_uint4(out[l][0], out[l][1], out[l][2], out[l][3]);
    }
    if (TALL) {
        __syncthreads();
#pragma unroll
        for (int l = 0; l < LIMBS; ++l)
            for (int e = threadIdx.x; e < OT_TILE / 16; e += 256)
                *reinterpret_cast<uint4*>(to + l * limb_bytes + e * 16) = *reinterpret_cast<const uint4*>(&s_tile[l][e * 16]);
    }
}

// ---- the products -----------------------------------------------------------------------------------------------------
struct OtGemm {
    const uint8_t* a;    // left operand's tiles [batch][limbs][rows / 128][a_width]
    const uint8_t* b;    // right operand's tiles [batch][limbs][rows / 128][b_width]
    uint8_t* out;        // the result's tiles [batch][limbs][rows / 128][out_width]
    int64_t a_limb, b_limb, out_limb;  // bytes of a limb
    int a_width, b_width, out_width;
    int chunks;          // of K, 64 each: what lies beyond them in the tiles is never read as K, whatever it holds
    int row_tiles;       // of the result
    int col_tiles;
    float ca, cb, cc;    // square: a I + b A + c A A
    float* part;         // Gram in gridDim.y parts of K: the parts' sums [batch][tile][part][32 column quads][128 rows][4]
};

template <int LIMBS>
struct OtShape {
    static constexpr int STAGE = LIMBS * 2 * OT_TILE;
    static constexpr int STAGES = LIMBS == 2 ? 3 : 6;
    static constexpr int SMEM = STAGE * STAGES + 1024;
    // chunks of 64 whose products share an accumulator (two limbs: four instead of one are 4 to 9 % faster and three times as far off, and a chunk's small products
    // have to be the first in what is scaled after them)
    static constexpr int DRAIN = LIMBS == 2 ? 1 : 1 << 30;
};

// a tile's place: of a symmetric result those on and below the diagonal, row by row
struct OtTile {
    int batch, i, j;
};
// W: columns of a tile, in 64s.  A tile of 64 or 128 columns has 128 rows, one of 256 has 256
template <int W>
__host__ __device__ constexpr int ot_sym_tiles(int row_tiles) { return W == 1 ? row_tiles * (row_tiles + 1) : row_tiles * (row_tiles + 1) / 2; }
template <bool SYM, int W>
__device__ __forceinline__ OtTile ot_tile(const OtGemm& g, int t, int tiles) {
    OtTile p;
    p.batch = t / tiles;
    t -= p.batch * tiles;
    if (SYM && W == 1) {
        p.i = (int)((sqrtf(4.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while ((p.i + 1) * (p.i + 2) <= t) ++p.i;
        while (p.i * (p.i + 1) > t) --p.i;
        p.j = t - p.i * (p.i + 1);
    } else if (SYM) {
        p.i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while ((p.i + 1) * (p.i + 2) / 2 <= t) ++p.i;
        while (p.i * (p.i + 1) / 2 > t) --p.i;
        p.j = t - p.i * (p.i + 1) / 2;
    } else {
        p.i = t % g.row_tiles;
        p.j = t / g.row_tiles;
    }
    return p;
}

__device__ __forceinline__ void ot_store_shared(uint8_t* p, __half v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(ot_smem(p)), "h"(__half_as_ushort(v)) : "memory");
}
__device__ __forceinline__ void ot_put(void* dst, unsigned src, unsigned bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

// 16 fp16 numbers of a row as they lie in a tile: two 16-byte pieces, which have changed places in odd rows
struct OtSector {
    unsigned w[8];
    __device__ __forceinline__ void load(const uint8_t* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 16);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
    __device__ __forceinline__ void exchange(int swap) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned a = w[i], b = w[i + 4];
            w[i] = swap ? b : a;
            w[i + 4] = swap ? a : b;
        }
    }
    __device__ __forceinline__ float get(int i) const { return op_word<__half>(w[i >> 1], i & 1); }
    // into a tile's image in shared memory, the first piece at that place of the row and the second at its neighbour
    __device__ __forceinline__ void store_shared(uint8_t* row, int place) const {
        const unsigned p = ot_smem(row);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p + (place << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p + ((place ^ 1) << 4)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    }
};

// W, a tile's columns in 64s.  W = 4: a cluster of two blocks computes 256 x 256 with cta_group::2 MMAs: each block holds 128 rows of the left
// operand, 128 columns of the right one and 128 x 256 accumulators; the even block issues the MMAs.  W = 2 and 1: a block computes 128 x 128 or
// 128 x 64.  Where all tiles run at once, half of a tile is half of its MMAs and of its epilogue: 359 x 785 170 us with 128 x 128 tiles, 127 with
// 128 x 64 (fp32; bf16 90 and 74), 65 x 65 92 and 68 us.
// Warps 0-7 read the accumulators (warp w: lanes 32 (w % 4) .. of them, columns 32 W (w / 4) ..), warp 8 copies, warp 9 issues the MMAs.
// MULTI: a block (pair) takes the tiles t, t + blocks, ..; while the eight warps store a tile from their registers, the next one's copies and MMAs are
// under way.  Those stores go straight to memory in whole 32-byte sectors (one instruction per lane; a tile's 16-byte pieces swap places inside their
// sector in odd rows), the mirrored tile's in 64 bytes per warp.  4096 x 4096 in bf16: 1406 us with a block per tile, 1200 so.  Where all tiles run at once
// they leave through shared memory, 5 % sooner, and both in one kernel would cost the small products 15 % (a launch runs through its code once).
template <int KIND, int LIMBS, int W, bool MULTI, typename T>
__global__ void __launch_bounds__(320, 1) k_orth_gemm(OtGemm g, OrthIo io) {
    using S = OtShape<LIMBS>;
    constexpr int CTAS = W == 4 ? 2 : 1;
    constexpr int TN = 64 * W, COLS = 32 * W;  // accumulator columns of a block, of a thread
    constexpr int HALF = OT_TILE / 2;          // 64 rows of a tile
    constexpr int RC = W == 1 ? 32 : 64;       // columns of a thread that leave at a time
    constexpr bool SYM = KIND == OT_GRAM || KIND == OT_SQUARE || KIND == OT_GRAM_PART;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) unsigned long long s_full[S::STAGES], s_peer[S::STAGES], s_empty[S::STAGES], s_acc_full[2], s_acc_empty[2];
    __shared__ __align__(8) unsigned long long s_quiet;  // this block's copies have landed and the pair's MMAs are done
    __shared__ unsigned s_tmem;
    uint8_t* s_dyn = s_raw + ((1024u - (ot_smem(s_raw) & 1023u)) & 1023u);
    const unsigned ring = ot_smem(s_dyn);
    // the warp's number is the same in its lanes, and the compiler has to know it: what the MMAs take lives in uniform registers then
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    const int tiles = SYM ? ot_sym_tiles<W>(g.row_tiles) : g.row_tiles * g.col_tiles, total = tiles * io.batch;
    const OtTile only = ot_tile<SYM, W>(g, first, tiles);  // of a block with one tile: known before the launch ahead is done
    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            ot_bar_init(ot_smem(&s_full[s]), 1);
            ot_bar_init(ot_smem(&s_peer[s]), 1);
            ot_bar_init(ot_smem(&s_empty[s]), 1);
        }
        for (int q = 0; q < 2; ++q) {
            ot_bar_init(ot_smem(&s_acc_full[q]), 1);
            ot_bar_init(ot_smem(&s_acc_empty[q]), 8 * CTAS);
        }
        ot_bar_init(ot_smem(&s_quiet), 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        if (CTAS == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ot_smem(&s_tmem)), "r"(2 * TN) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ot_smem(&s_tmem)), "r"(2 * TN) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CTAS == 2) ot_cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    op_wait_for_previous();
    op_next_may_start();
    const unsigned tmem = s_tmem;
    const int chunk0 = KIND == OT_GRAM_PART ? (int)((int64_t)g.chunks * blockIdx.y / gridDim.y) : 0;
    const int chunks = KIND == OT_GRAM_PART ? (int)((int64_t)g.chunks * (blockIdx.y + 1) / gridDim.y) - chunk0 : g.chunks;
    const int rounds = (chunks + S::DRAIN - 1) / S::DRAIN;
    bool ok = true;

    if (warp == 8) {
        asm volatile("fence.proxy.async;" ::: "memory");  // bulk copies read what the launch ahead has stored
        unsigned s = 0, parity = 1;  // a barrier that nothing has arrived at yet passes for the phase before its first
        int64_t count = 0;           // chunks issued
        for (int t = first; ok && t < total; t += MULTI ? step : total) {
            const OtTile at = MULTI ? ot_tile<SYM, W>(g, t, tiles) : only;
            const bool same = SYM && at.i == (W == 1 ? at.j >> 1 : at.j);
            const int col_tile = at.j * CTAS + rank;  // this block's columns of the right operand, in 128s (W = 1: 64s)
            const uint8_t* a = g.a + (int64_t)at.batch * LIMBS * g.a_limb + ((int64_t)(at.i * CTAS + rank) * g.a_width + chunk0) * OT_TILE;
            // SYM: the tiles of a row, one after the other; else two half tiles (64 rows) at a time, the next rows' half in the same tiles or a row of tiles on
            const uint8_t* b = g.b + (int64_t)at.batch * LIMBS * g.b_limb + (W == 1 ? (SYM ? ((int64_t)(col_tile >> 1) * g.b_width + chunk0) * OT_TILE + (col_tile & 1) * HALF : (int64_t)col_tile * OT_TILE)
                                                                                : (SYM ? (int64_t)col_tile * g.b_width + chunk0 : (int64_t)2 * col_tile) * OT_TILE);
            const int64_t b_odd = SYM ? OT_TILE : HALF, b_even = SYM ? OT_TILE : (int64_t)g.b_width * OT_TILE - HALF;
            const unsigned bytes = LIMBS * (same ? OT_TILE : W == 1 ? OT_TILE + HALF : 2 * OT_TILE);
            for (int k = 0; k < chunks; ++k, ++count) {
                const unsigned bar = ot_smem(&s_full[0]) + 8 * s, to = ring + s * S::STAGE;
                ok = __all_sync(0xffffffffu, ot_wait<OT_COPIES>(ot_smem(&s_empty[0]) + 8 * s, parity));
                if (!ok) break;
                if (lane == 0) {
                    ot_expect(bar, bytes);
#pragma unroll
                    for (int l = 0; l < LIMBS; ++l) {
                        ot_copy(to + l * OT_TILE, a + l * g.a_limb, OT_TILE, bar);
                        if (same) continue;
                        const unsigned tb = to + (LIMBS + l) * OT_TILE;
                        ot_copy(tb, b + l * g.b_limb, SYM && W > 1 ? OT_TILE : HALF, bar);
                        if (!SYM && W > 1) ot_copy(tb + HALF, b + l * g.b_limb + OT_TILE, HALF, bar);
                    }
                }
                __syncwarp();
                a += OT_TILE;
                b += k & 1 ? b_even : b_odd;
                if (++s == S::STAGES) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
        // whoever gave up: the copies land before the block ends
        for (int64_t q = count < S::STAGES ? 0 : count - S::STAGES; q < count; ++q) ot_wait<OT_END>(ot_smem(&s_full[q % S::STAGES]), (unsigned)((q / S::STAGES) & 1));
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ot_smem(&s_quiet)) : "memory");
    } else if (warp == 9) {
        unsigned s = 0, parity = 0;
        if (rank == 0) {
            // fp32 accumulator (1 at bit 4), fp16 operands, N / 8 at bit 17, M / 16 at bit 24; apply: the right operand is N-major (bit 16)
            constexpr unsigned IDESC = (1u << 4) | (SYM ? 0u : 1u << 16) | ((unsigned)(TN / 8) << 17) | ((unsigned)(8 * CTAS) << 24);
            // descriptors of the first stage; steps along K and to other stages are added in units of 16 bytes.  K-major: 32 bytes along the
            // row, 8-row groups 1024 bytes apart.  N-major: 16 rows of 128 bytes, 8-row groups 1024 bytes apart, the next 64 columns 8 KB further
            const unsigned long long da0 = ot_desc(ring, 16, 1024);
            constexpr unsigned STEP_A = 2, STEP_B = SYM ? 2 : 128;
            const bool leader = ot_elect();
            unsigned buffer = 0, drained = 1;  // the accumulator, and the parity of its being empty
            for (int t = first; ok && t < total; t += MULTI ? step : total) {
                const OtTile at = MULTI ? ot_tile<SYM, W>(g, t, tiles) : only;
                const bool same = SYM && at.i == (W == 1 ? at.j >> 1 : at.j);
                const unsigned b_at = same ? ring + (W == 1 ? (at.j & 1) * HALF : 0) : ring + LIMBS * OT_TILE;
                const unsigned long long db0 = SYM ? ot_desc(b_at, 16, 1024) : ot_desc(b_at, HALF, 1024);
                int k = 0;
                for (int r = 0; r < rounds && ok; ++r) {
                    const unsigned d = tmem + buffer * TN;
                    ok = __all_sync(0xffffffffu, ot_wait<OT_PRODUCTS>(ot_smem(&s_acc_empty[0]) + 8 * buffer, drained));
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int last = min(chunks, k + S::DRAIN);
                    unsigned accumulate = 0;
                    for (; ok && k < last; ++k) {
                        ok = ot_wait<OT_PRODUCTS>(ot_smem(&s_full[0]) + 8 * s, parity);
                        if (CTAS == 2) ok = ok && ot_wait<OT_PRODUCTS>(ot_smem(&s_peer[0]) + 8 * s, parity);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (leader) {
                            const unsigned long long da = da0 + s * (S::STAGE / 16), db = db0 + s * (S::STAGE / 16);
#pragma unroll
                            for (int q = 0; q < (LIMBS == 2 ? 3 : 1); ++q)  // high low, low high, high high: the large terms last
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const unsigned long long a = da + (LIMBS == 2 && q == 1 ? OT_TILE / 16 : 0) + STEP_A * j, b = db + (LIMBS == 2 && q == 0 ? OT_TILE / 16 : 0) + STEP_B * j;
                                    const unsigned more = q > 0 || j > 0 ? 1u : accumulate;
                                    if (q == 2 && j == 0) ot_mma<CTAS, OT_LOW_BITS>(d, a, b, IDESC, more);
                                    else ot_mma<CTAS, 0>(d, a, b, IDESC, more);
                                }
                            ot_commit<CTAS>(ot_smem(&s_empty[0]) + 8 * s);
                        }
                        __syncwarp();
                        accumulate = 1;
                        if (++s == S::STAGES) {
                            s = 0;
                            parity ^= 1;
                        }
                    }
                    if (leader && ok) ot_commit<CTAS>(ot_smem(&s_acc_full[0]) + 8 * buffer);
                    __syncwarp();
                    drained ^= buffer;
                    buffer ^= 1;
                }
            }
            if (leader) ot_commit<CTAS>(ot_smem(&s_quiet));
        } else {
            // the odd block: tells the even one that its operands are there
            for (int t = first; ok && t < total; t += MULTI ? step : total)
                for (int k = 0; k < chunks && ok; ++k) {
                    ok = __all_sync(0xffffffffu, ot_wait<OT_RELAY>(ot_smem(&s_full[0]) + 8 * s, parity));
                    if (ok && lane == 0) ot_arrive_at(ot_smem(&s_peer[0]) + 8 * s, 0);
                    __syncwarp();
                    if (++s == S::STAGES) {
                        s = 0;
                        parity ^= 1;
                    }
                }
        }
        ot_wait<OT_END>(ot_smem(&s_quiet), 0);
    } else {
        const unsigned taddr = tmem + ((unsigned)((warp & 3) * 32) << 16) + (unsigned)((warp >> 2) * COLS);
        const int group = warp >> 2, row = tid & 127;
        unsigned buffer = 0, filled = 0;
        for (int t = first; t < total; t += MULTI ? step : total) {
            const OtTile at = MULTI ? ot_tile<SYM, W>(g, t, tiles) : only;
            float acc[COLS];
#pragma unroll
            for (int c = 0; c < COLS; ++c) acc[c] = 0.0f;
            for (int r = 0; r < rounds && ok; ++r) {
                ok = __all_sync(0xffffffffu, ot_wait<OT_SUMS>(ot_smem(&s_acc_full[0]) + 8 * buffer, filled));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c0 = 0; c0 < COLS; c0 += 32) {
                    unsigned v[32];
                    ot_read32(taddr + buffer * TN + c0, v);
#pragma unroll
                    for (int c = 0; c < 32; ++c) acc[c0 + c] += __uint_as_float(v[c]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 2) ot_arrive_at(ot_smem(&s_acc_empty[0]) + 8 * buffer, 0);
                    else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ot_smem(&s_acc_empty[0]) + 8 * buffer) : "memory");
                }
                filled ^= buffer;
                buffer ^= 1;
            }
            if (!ok) {
                ot_wait<OT_END>(ot_smem(&s_quiet), 0);  // what is stored may pass through the ring
#pragma unroll
                for (int c = 0; c < COLS; ++c) acc[c] = __int_as_float(0x7fc00000);
            }

            if (KIND == OT_GRAM_PART) {
                static_assert(KIND != OT_GRAM_PART || W == 1, "parts are of tiles of 64 columns");
                const int whole = at.batch * (tiles / 2) + at.i * (at.i + 1) / 2 + (at.j >> 1), from = (at.j & 1) * 64;  // in the 128 x 128 tiles
                float4* to = reinterpret_cast<float4*>(g.part) + ((int64_t)whole * gridDim.y + blockIdx.y) * 4096 + row;
#pragma unroll
                for (int c = 0; c < COLS; c += 4) to[(from + group * COLS + c) / 4 * 128] = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
            } else if (KIND == OT_LAST && MULTI && io.rows > io.cols) {
                // rows of X are columns of the result: a warp's lanes are neighbours there.  Eight old weights on their way
                const int i = (at.i * CTAS + rank) * 128 + row, j0 = (at.j * 2 + group) * COLS, left = io.rows - j0;
                int64_t to = at.batch * io.out_batch + j0 * io.out_stride + i;
                if (i < io.cols)
#pragma unroll
                    for (int c0 = 0; c0 < COLS; c0 += 8, to += 8 * io.out_stride) {
                        if (c0 >= left) break;
                        if (!io.m) {
                            T* out = static_cast<T*>(io.out) + to;
#pragma unroll
                            for (int c = 0; c < 8; ++c, out += io.out_stride)
                                if (c0 + c < left) *out = op_round<T>(acc[c0 + c] * OT_UNSCALE);
                            continue;
                        }
                        float w[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) w[c] = c0 + c < left ? io.w[to + c * io.out_stride] : 0.0f;
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (c0 + c < left) static_cast<float*>(io.out)[to + c * io.out_stride] = orth_update(io, w[c], acc[c0 + c] * OT_UNSCALE);
                    }
            } else if (KIND == OT_LAST && MULTI) {
                // rows on 16-byte boundaries go out straight from the registers, eight elements at a time
                const int i = (at.i * CTAS + rank) * 128 + row, j0 = (at.j * 2 + group) * COLS;
                const int64_t to = at.batch * io.out_batch + i * io.out_stride + j0;
                if (i < io.rows)
#pragma unroll
                    for (int c0 = 0; c0 < COLS; c0 += 8) {
                        if (j0 + c0 >= io.cols) break;  // a multiple of eight
                        float x[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) x[c] = acc[c0 + c] * OT_UNSCALE;
                        if (io.m) {
                            float w[2][4];
#pragma unroll
                            for (int h = 0; h < 2; ++h) op_load<float, 4>(io.w + to + c0 + 4 * h, w[h]);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float q[4];
#pragma unroll
                                for (int c = 0; c < 4; ++c) q[c] = orth_update(io, w[h][c], x[4 * h + c]);
                                op_store<float, 4>(static_cast<float*>(io.out) + to + c0 + 4 * h, q);
                            }
                        } else {
                            constexpr int STEP = 16 / (int)sizeof(T);
#pragma unroll
                            for (int h = 0; h < 8; h += STEP) {
                                float q[STEP];
#pragma unroll
                                for (int c = 0; c < STEP; ++c) q[c] = x[h + c];
                                op_store<T, STEP>(static_cast<T*>(io.out) + to + c0 + h, q);
                            }
                        }
                    }
            } else if (KIND == OT_LAST) {
                // rows that start anywhere: by rounds of 64 (W = 1: 32) columns through shared memory (a block has one tile, its ring is free by now)
                float* flat = reinterpret_cast<float*>(s_dyn + group * 40960);  // [128][65]
#pragma unroll
                for (int h = 0; h < CTAS; ++h) {
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
#pragma unroll
                    for (int c = 0; c < RC; ++c) flat[row * 65 + c] = acc[RC * h + c] * OT_UNSCALE;
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
                    const int i0 = (at.i * CTAS + rank) * 128, j0 = W == 1 ? at.j * 64 + group * 32 : (at.j * 2 * CTAS + group * CTAS + h) * 64;
                    // 64 (32) neighbours of two (four) rows at a time, eight of a thread's old weights on their way
                    constexpr int AT_ONCE = 128 / RC;
                    const int r = row / RC, c = row % RC;
                    const int64_t to = at.batch * io.out_batch + (i0 + r) * io.out_stride + j0 + c, next = AT_ONCE * io.out_stride;
                    const int left = j0 + c < io.cols ? (io.rows - i0 - r + AT_ONCE - 1) / AT_ONCE : 0;
                    const float* from = flat + r * 65 + c;
                    for (int e0 = 0; e0 < RC && e0 < left; e0 += 8) {
                        float w[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) w[u] = io.m && e0 + u < left ? io.w[to + (e0 + u) * next] : 0.0f;
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            if (e0 + u < left) orth_store<T>(io, to + (e0 + u) * next, w[u], from[(e0 + u) * 65 * AT_ONCE]);
                    }
                }
            } else {
                const bool same = SYM && at.i == (W == 1 ? at.j >> 1 : at.j);
                const int row_tile = at.i * CTAS + rank;
                uint8_t* out = g.out + (int64_t)at.batch * LIMBS * g.out_limb;
                // Nothing follows a block's only tile, so its ring is free for images of the result's tiles, which go out as bulk copies.  An image:
                // [limb] tile, then mirrored [limb][column half] half a tile of 64 rows; every round has its own where the ring has room.
                constexpr bool staged = !MULTI;
                constexpr int IMAGES = (SYM ? 2 : 1) * LIMBS * OT_TILE;
                constexpr bool APART = 2 * CTAS * IMAGES <= S::STAGE * S::STAGES;
                const int swap = row & 1;  // of a sector's two pieces
                const float square = g.cc * (OT_UNSCALE * OT_SCALE);
#pragma unroll
                for (int h = 0; h < CTAS; ++h) {
                    const int col_tile = W == 1 ? at.j : at.j * 2 * CTAS + group * CTAS + h;  // the round's columns, in 64s
                    const int base = W == 1 ? group * 32 : 0;                               // W = 1: both groups have half of the same ones
                    const int64_t to_direct = ((int64_t)row_tile * g.out_width + col_tile) * OT_TILE;
                    const int64_t to_mirror = ((int64_t)(col_tile >> 1) * g.out_width + 2 * row_tile) * OT_TILE + (col_tile & 1) * (OT_TILE / 2);
                    uint8_t* image = s_dyn + (W == 1 ? 0 : group + (APART ? 2 * h : 0)) * IMAGES;
                    uint8_t* direct = staged ? image + row * 128 : out + to_direct + row * 128;
                    const int64_t direct_limb = staged ? OT_TILE : g.out_limb;
                    uint8_t* mirror = staged ? image + LIMBS * OT_TILE + (row >> 6) * (OT_TILE / 2) + (row & 7) * 2 : out + to_mirror + (row >> 6) * OT_TILE + (row & 7) * 2;
                    const uint8_t* old = g.a + (int64_t)at.batch * LIMBS * g.a_limb + ((int64_t)row_tile * g.a_width + col_tile) * OT_TILE + row * 128;
                    const int ident = row_tile * 128 + row - col_tile * 64 - base;  // the diagonal's column
                    if (h && staged && !APART) asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
                    OtSector before[LIMBS];  // square: A, a sector ahead
                    if (KIND == OT_SQUARE)
#pragma unroll
                        for (int l = 0; l < LIMBS; ++l) before[l].load(old + l * g.a_limb + (((base >> 3) ^ (row & 6)) << 4));
#pragma unroll
                    for (int c0 = 0; c0 < RC; c0 += 16) {
                        float x[16];  // scaled as it is stored
#pragma unroll
                        for (int c = 0; c < 16; ++c) x[c] = acc[RC * h + c0 + c] * (KIND == OT_SQUARE ? square : OT_UNSCALE * OT_SCALE);
                        if (KIND == OT_SQUARE) {
#pragma unroll
                            for (int l = LIMBS - 1; l >= 0; --l) {
                                before[l].exchange(swap);
#pragma unroll
                                for (int c = 0; c < 16; ++c) x[c] = fmaf(l ? g.cb / OT_LOW : g.cb, before[l].get(c), x[c]);
                                if (c0 + 16 < RC) before[l].load(old + l * g.a_limb + ((((base + c0 + 16) >> 3) ^ (row & 6)) << 4));
                            }
                            if (same)  // the diagonal passes through these tiles alone
#pragma unroll
                                for (int c = 0; c < 16; ++c) x[c] += ident == c0 + c ? g.ca * OT_SCALE : 0.0f;
                        }
                        OtSector piece[LIMBS];
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            __half2 pair[LIMBS];
                            ot_split<LIMBS>(x[c], x[c + 1], pair);
#pragma unroll
                            for (int l = 0; l < LIMBS; ++l) {
                                piece[l].w[c / 2] = *reinterpret_cast<const unsigned*>(&pair[l]);
                                if (SYM && !same) {
                                    uint8_t* to = mirror + (staged ? l * OT_TILE : l * g.out_limb) + (base + c0 + c) * 128;
                                    const int slot = (row & 63) >> 3;
                                    if (staged) {  // not left to the compiler: a generic store costs as much as a global one
                                        ot_store_shared(to + (((slot ^ (c0 + c)) & 7) << 4), __low2half(pair[l]));
                                        ot_store_shared(to + 128 + (((slot ^ (c0 + c + 1)) & 7) << 4), __high2half(pair[l]));
                                    } else {
                                        *reinterpret_cast<__half*>(to + (((slot ^ (c0 + c)) & 7) << 4)) = __low2half(pair[l]);
                                        *reinterpret_cast<__half*>(to + 128 + (((slot ^ (c0 + c + 1)) & 7) << 4)) = __high2half(pair[l]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int l = 0; l < LIMBS; ++l) {
                            uint8_t* to = direct + l * direct_limb;
                            if (staged) {
                                piece[l].store_shared(to, ((base + c0) >> 3) ^ (row & 7));
                            } else {
                                piece[l].exchange(swap);
                                piece[l].store(to + ((((base + c0) >> 3) ^ (row & 6)) << 4));
                            }
                        }
                    }
                    if (staged) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        if (W == 1) asm volatile("bar.sync 1, 256;" ::: "memory");
                        else asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
                        if (W == 1 ? tid == 0 : row == 0) {
#pragma unroll
                            for (int l = 0; l < LIMBS; ++l) {
                                ot_put(out + l * g.out_limb + to_direct, ot_smem(image + l * OT_TILE), OT_TILE);
                                if (SYM && !same) {
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        ot_put(out + l * g.out_limb + to_mirror + q * OT_TILE, ot_smem(image + (LIMBS + l) * OT_TILE + q * (OT_TILE / 2)), OT_TILE / 2);
                                }
                            }
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                            // the images must be read before they are written again, or the block ends
                            if (!APART || h + 1 == CTAS) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CTAS == 2) ot_cluster_sync();  // the other block's MMAs are done with this block's memory, and no signal is under way
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 9) {
        if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TN) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TN) : "memory");
    }
}

// The parts of a Gram matrix, added in order, as tiles: eight columns of a tile per block.
template <int LIMBS>
__global__ void __launch_bounds__(256) k_orth_join(const float* __restrict__ part, int parts, uint8_t* __restrict__ out, int64_t limb_bytes, int width) {
    const int tile = blockIdx.x >> 4, batch = blockIdx.z, tiles = gridDim.x >> 4;
    int ti = 0;
    while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
    const int tj = tile - ti * (ti + 1) / 2, row = threadIdx.x & 127, quad = (blockIdx.x & 15) * 2 + (threadIdx.x >> 7), col = quad * 4;
    op_wait_for_previous();
    op_next_may_start();
    const float4* p = reinterpret_cast<const float4*>(part) + ((int64_t)batch * tiles + tile) * parts * 4096 + quad * 128 + row;
    float4 t[OT_PARTS];
#pragma unroll
    for (int q = 0; q < OT_PARTS; ++q) t[q] = q < parts ? p[(int64_t)q * 4096] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float x[4] = {t[0].x, t[0].y, t[0].z, t[0].w};
#pragma unroll
    for (int q = 1; q < OT_PARTS; ++q) {
        x[0] += t[q].x;
        x[1] += t[q].y;
        x[2] += t[q].z;
        x[3] += t[q].w;
    }
    uint8_t* o = out + (int64_t)batch * LIMBS * limb_bytes;
    OpVec<__half, 4> piece[LIMBS];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        __half s[LIMBS];
        ot_split<LIMBS>(x[c] * (OT_UNSCALE * OT_SCALE), s);
#pragma unroll
        for (int l = 0; l < LIMBS; ++l) {
            piece[l].v[c] = s[l];
            if (ti != tj) *reinterpret_cast<__half*>(o + l * limb_bytes + ((int64_t)tj * width + 2 * ti + (row >> 6)) * OT_TILE + ot_at(col + c, row & 63)) = s[l];
        }
    }
#pragma unroll
    for (int l = 0; l < LIMBS; ++l)
        *reinterpret_cast<OpVec<__half, 4>*>(o + l * limb_bytes + ((int64_t)ti * width + 2 * tj + (col >> 6)) * OT_TILE + ot_at(row, col & 63)) = piece[l];
}

struct OtPlan {
    int sym, all;                            // columns of a tile of the symmetric products and of Q X, in 64s
    int parts;                               // of K in the Gram product
    int n, m;
    int64_t n_pad, m_pad;
    int64_t x_limb, a_limb;                  // bytes of a limb
    int64_t x0, x1, a, q, part, total;       // offsets in the workspace
};
// Cycles of a product by the waves of its tiles: a chunk of K in a tile of 64, 128 (one block) or 256 (two) columns, with one limb or two, and
// a tile's fixed part (launch, first copies, epilogue), as measured at n = 777, m = 1000 and 4096 x 4096 and, for 64 columns, n = 359, m = 785.
int64_t ot_chunk(int limbs, int w) { return limbs == 1 ? (w == 1 ? 350 : w == 2 ? 390 : 450) : w == 1 ? 600 : w == 2 ? 990 : 1520; }
int64_t ot_cost(int64_t tiles, int64_t chunks, int limbs, int w) {
    const int64_t slots = sm_count() / (w == 4 ? 2 : 1), waves = (tiles + slots - 1) / slots;
    return waves * (chunks * ot_chunk(limbs, w) + (w == 1 ? 8000 : w == 2 ? 9000 : limbs == 1 ? 13000 : 18000));
}
OtPlan ot_plan(int batch, int rows, int cols, int limbs) {
    OtPlan p;
    p.n = rows < cols ? rows : cols;
    p.m = rows < cols ? cols : rows;
    const int64_t n = p.n, m = p.m;  // m + 255 may be beyond 2^31
    const int64_t n1 = (n + 127) / 128, n2 = (n + 255) / 256, m1 = (m + 127) / 128, m2 = (m + 255) / 256, kn = (n + 63) / 64, km = (m + 63) / 64;
    int64_t best = 0, sym_best = 0;
    for (int w = 1; w <= 4; w *= 2) {
        const int64_t sym = batch * (w == 4 ? n2 * (n2 + 1) / 2 : n1 * (n1 + 1) / (w == 1 ? 1 : 2)), all = batch * (w == 4 ? n2 * m2 : w == 2 ? n1 * m1 : 2 * n1 * m1);
        const int64_t cs = ot_cost(sym, kn, limbs, w) + ot_cost(sym, km, limbs, w), ca = ot_cost(all, kn, limbs, w);
        if ((w > 1 || sym <= sm_count()) && (sym_best == 0 || cs < sym_best)) sym_best = cs, p.sym = w;
        if ((w > 1 || all <= sm_count()) && (best == 0 || ca < best)) best = ca, p.all = w;
    }
    // few tiles with a long K are cut into parts where that saves more than the launch that joins them
    p.parts = 1;
    const int64_t s1 = batch * n1 * (n1 + 1) / 2;
    if (p.sym == 1) {  // room for another part of 128 x 128 tiles is room for tiles of half the size
        int64_t q = sm_count() / (2 * s1);
        q = q < OT_PARTS ? q : OT_PARTS;
        q = q < km / 4 ? q : km / 4;
        if (q > 1 && (km - km / q) * ot_chunk(limbs, 1) > 9000) p.parts = (int)q;
    }
    const int pad = p.sym == 4 || p.all == 4 ? 256 : 128;
    p.n_pad = (n + pad - 1) / pad * pad;
    p.m_pad = (m + pad - 1) / pad * pad;
    p.x_limb = p.n_pad * p.m_pad * 2;
    p.a_limb = p.n_pad * p.n_pad * 2;
    p.x0 = ((int64_t)batch * OT_NORM_BLOCKS * 8 + 127) / 128 * 128;
    p.x1 = p.x0 + p.x_limb * limbs * batch;
    p.a = p.x1 + p.x_limb * limbs * batch;
    p.q = p.a + p.a_limb * limbs * batch;
    p.part = p.q + p.a_limb * limbs * batch;
    p.total = p.part + (p.parts > 1 ? s1 * p.parts * 65536 : 0);
    return p;
}

template <int KIND, int LIMBS, int W, bool MULTI, typename T>
void ot_launch(cudaStream_t s, const OtGemm& g, const OrthIo& io, int64_t blocks, int parts) {
    using S = OtShape<LIMBS>;
    constexpr int CTAS = W == 4 ? 2 : 1;
    auto kern = k_orth_gemm<KIND, LIMBS, W, MULTI, T>;
    static std::atomic<uint64_t> known{0};  // devices on which the kernel may take that much shared memory
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !(known.load(std::memory_order_relaxed) >> dev & 1)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e == cudaSuccess && dev >= 0 && dev < 64) known.fetch_or(1ull << dev);
        op_note(e);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * CTAS), (unsigned)parts);
    cfg.blockDim = dim3(320);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CTAS;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CTAS == 2 ? 2 : 1;
    op_note(cudaLaunchKernelEx(&cfg, kern, g, io));
}
template <int KIND, int LIMBS, int W, typename T>
void ot_gemm_of(cudaStream_t s, const OtGemm& g, const OrthIo& io, int parts) {
    const int64_t tiles = KIND == OT_APPLY || KIND == OT_LAST ? (int64_t)g.row_tiles * g.col_tiles : ot_sym_tiles<W>(g.row_tiles);
    const int64_t all = tiles * io.batch, slots = sm_count() / (W == 4 ? 2 : 1);
    if constexpr (KIND == OT_LAST) {  // MULTI: the result can be stored straight from the registers
        const bool aligned = io.cols % 8 == 0 && io.out_stride % 8 == 0 && io.out_batch % 8 == 0 && (((uintptr_t)io.out | (uintptr_t)io.w) & 15) == 0;
        if (io.rows > io.cols || aligned) return ot_launch<KIND, LIMBS, W, true, T>(s, g, io, all > slots ? slots : all, parts);
    } else if constexpr (KIND != OT_GRAM_PART && W > 1) {  // tiles of 64 columns are taken where all run at once
        if (all > slots) return ot_launch<KIND, LIMBS, W, true, T>(s, g, io, slots, parts);
    }
    ot_launch<KIND, LIMBS, W, false, T>(s, g, io, all, parts);
}
template <int KIND, int LIMBS, typename T>
void ot_gemm(cudaStream_t s, const OtGemm& g, const OrthIo& io, int w, int parts = 1) {
    if constexpr (KIND == OT_GRAM_PART) return ot_gemm_of<KIND, LIMBS, 1, T>(s, g, io, parts);
    else if (w == 1) ot_gemm_of<KIND, LIMBS, 1, T>(s, g, io, parts);
    else if (w == 2) ot_gemm_of<KIND, LIMBS, 2, T>(s, g, io, parts);
    else ot_gemm_of<KIND, LIMBS, 4, T>(s, g, io, parts);
}

template <typename T, int LIMBS>
void ot_steps(cudaStream_t s, const OrthIo& io, const OrthPoly& poly, uint8_t* work, const OtPlan& p) {
    uint8_t *x = work + p.x0, *y = work + p.x1, *a = work + p.a, *q = work + p.q;
    const int wn = (int)(p.n_pad / 64), wm = (int)(p.m_pad / 64), kn = (int)ceil_div64(p.n, 64), km = (int)ceil_div64(p.m, 64);
    const int sym_rows = p.sym == 4 ? 256 : 128, all_rows = p.all == 4 ? 256 : 128;
    const int st = (int)ceil_div64(p.n, sym_rows), rt = (int)ceil_div64(p.n, all_rows), ct = (int)ceil_div64(p.m, all_rows) * (p.all == 1 ? 2 : 1);
    float* part = reinterpret_cast<float*>(work + p.part);
    for (int k = 0; k < poly.steps; ++k) {
        const OtGemm gram = {x, x, a, p.x_limb, p.x_limb, p.a_limb, wm, wm, wn, km, st, st, 0.f, 0.f, 0.f, part};
        const OtGemm square = {a, a, q, p.a_limb, p.a_limb, p.a_limb, wn, wn, wn, kn, st, st, poly.a, poly.b, poly.c, nullptr};
        const OtGemm apply = {q, x, y, p.a_limb, p.x_limb, p.x_limb, wn, wm, wm, kn, rt, ct, 0.f, 0.f, 0.f, nullptr};
        if (p.parts > 1) {
            ot_gemm<OT_GRAM_PART, LIMBS, float>(s, gram, io, p.sym, p.parts);
            op_launch_next(s, dim3((unsigned)(st * (st + 1) / 2 * 16), 1, (unsigned)io.batch), dim3(256), 0, k_orth_join<LIMBS>, part, p.parts, a, p.a_limb, wn);
        } else {
            ot_gemm<OT_GRAM, LIMBS, float>(s, gram, io, p.sym);
        }
        ot_gemm<OT_SQUARE, LIMBS, float>(s, square, io, p.sym);
        if (k + 1 < poly.steps) ot_gemm<OT_APPLY, LIMBS, float>(s, apply, io, p.all);
        else ot_gemm<OT_LAST, LIMBS, T>(s, apply, io, p.all);
        uint8_t* z = x;
        x = y;
        y = z;
    }
}

// the norm and the tiles of X0; N: adjacent elements per access
template <typename T, int LIMBS, int N, bool MUON>
void ot_begin_of(cudaStream_t s, const OrthIo& io, const OrthPoly& poly, const OtPlan& p, double* partial, uint8_t* x) {
    const bool gaps = io.g_stride != io.cols;
    const int64_t total = gaps ? 0 : (int64_t)io.rows * io.cols, len = gaps ? io.cols : 4096, segments = gaps ? io.rows : (total + 4095) / 4096;
    int64_t most = 8 * (int64_t)sm_count() / io.batch;
    most = most < 1 ? 1 : most < OT_NORM_BLOCKS ? most : OT_NORM_BLOCKS;
    const int blocks = (int)(segments < most ? segments : most);
    // a matrix without gaps is read 16 bytes at a time even where its rows do not start on such a boundary
    constexpr int W = 16 / (int)sizeof(T);
    const bool flat = !gaps && total % W == 0 && ((uintptr_t)io.g & 15) == 0 && io.g_batch % W == 0 && (((uintptr_t)io.m | (uintptr_t)io.m_out) & 15) == 0;
    const dim3 grid0((unsigned)blocks, (unsigned)io.batch);
    op_launch_next(s, grid0, dim3(256), 0, flat ? k_orth_norm<T, W, MUON> : k_orth_norm<T, N, MUON>, io, segments, len, total, partial);
    const dim3 grid((unsigned)(p.m_pad / 64), (unsigned)(p.n_pad / 128), (unsigned)io.batch);
    if (io.rows > io.cols) op_launch_next(s, grid, dim3(256), 0, k_orth_pack<T, LIMBS, 1, true, MUON>, io, poly.eps, partial, blocks, x, p.x_limb);
    else op_launch_next(s, grid, dim3(256), 0, k_orth_pack<T, LIMBS, N, false, MUON>, io, poly.eps, partial, blocks, x, p.x_limb);
}

template <typename T, int LIMBS, int N>
void ot_begin(cudaStream_t s, const OrthIo& io, const OrthPoly& poly, const OtPlan& p, double* partial, uint8_t* x) {
    if constexpr (LIMBS == 2)  // Muon's update always has two
        if (io.m) return ot_begin_of<T, LIMBS, N, true>(s, io, poly, p, partial, x);
    ot_begin_of<T, LIMBS, N, false>(s, io, poly, p, partial, x);
}

template <typename T, int LIMBS>
void ot_run(cudaStream_t s, const OrthIo& io, const OrthPoly& poly, uint8_t* work) {
    const OtPlan p = ot_plan(io.batch, io.rows, io.cols, LIMBS);
    double* partial = reinterpret_cast<double*>(work);
    // 16 bytes at a time where all rows start on such a boundary
    constexpr int W = 16 / (int)sizeof(T);
    const bool wide = io.cols % W == 0 && ((uintptr_t)io.g & 15) == 0 && io.g_stride % W == 0 && io.g_batch % W == 0 && (((uintptr_t)io.m | (uintptr_t)io.m_out) & 15) == 0;
    if (wide) ot_begin<T, LIMBS, W>(s, io, poly, p, partial, work + p.x0); else ot_begin<T, LIMBS, 1>(s, io, poly, p, partial, work + p.x0);
    ot_steps<T, LIMBS>(s, io, poly, work, p);
}

}  // namespace

int64_t orth_tc_workspace(int batch, int rows, int cols, int limbs) { return ot_plan(batch, rows, cols, limbs).total; }

void launch_orth_tc(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int type, int limbs, void* work) {
    uint8_t* w = static_cast<uint8_t*>(work);
    if (type == TB_TYPE_F32) ot_run<float, 2>(s, io, p, w);
    else if (type == TB_TYPE_F16) ot_run<__half, 2>(s, io, p, w);
    else if (limbs == 2) ot_run<__nv_bfloat16, 2>(s, io, p, w);
    else ot_run<__nv_bfloat16, 1>(s, io, p, w);
}
