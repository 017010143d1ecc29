// Rows to the experts that a router chose for them, and back, on the caller's device tensors.
//
//   order      a stable sort of the choices [rows, k] by expert (op_sort.cuh): position, the place of every choice; source, the choice of every place;
//              offsets, where every expert's places begin.  A choice outside [0, experts) has no place, a place without a choice has source -1
//   dispatch   out[position[r, j]] = x[r];  rows of zeros at the places without a choice.  Its gradient is the combination without gates
//   combine    out[r] = sum over j of gate[r, j] * y[position[r, j]]
//   gradient   dy[position[r, j]] = gate[r, j] * dout[r],  dgate[r, j] = <dout[r], y[position[r, j]]>;  zeros at the places without a choice
//
// All are bound by memory: rows go by the order of the tokens, so a token's row is read once for all of its places; the places' rows are read or written
// once each, wherever they lie, in whole 16-byte accesses.  A group of lanes takes a row or a tile of its columns.  Sums are fp32: the choices in ascending order; a
// dot product's columns per thread in ascending order, then halves of the lanes, then the warps in order.
//
// Measured: dispatch 65536 x 1536 bf16 to two places each 95.5 us (6.3 TB/s); combination of 30011 x 1000 fp16 from eight places each 88 us (5.9 TB/s: gathers of 2000 bytes), its gradient for
// 40000 x 768 fp32 and two places 95.5 us (6.4 TB/s); the order of 65536 x 2 choices of 9 6 us, of 40000 x 8 of 256 15.6 us (launches that wait for one another).
#include "op_sort.cuh"

namespace {

#define EXPERT_MAX_K 16

struct ExpertSource {
    const int* index;
    __device__ __forceinline__ int operator()(int64_t i) const { return index[i]; }
    __device__ __forceinline__ int id(int64_t i) const { return (int)i; }
    __device__ __forceinline__ int key(int v) const { return v; }
};
struct ExpertPut {
    int *position, *source, *offsets;
    int64_t slots;
    __device__ __forceinline__ void operator()(int i, int, int place) const {
        position[i] = place;
        if (place >= 0) source[place] = i;
    }
    // the begins, and -1 at every place that no choice has taken
    __device__ __forceinline__ void rest(const int* total, const int* begin, const SortPlan& p) const {
        if (blockIdx.x == 0)
            for (int e = threadIdx.x; e <= p.keys; e += SORT_THREADS) offsets[e] = begin[e];
        // experts that have not filled their last `align` places: one for each warp of the launch in turn, looked at 32 at once
        const int lane = threadIdx.x & 31, warps = gridDim.x * SORT_WARPS;
        for (int e0 = blockIdx.x * SORT_WARPS + threadIdx.x / 32; e0 < p.keys && p.align > 1; e0 += 32 * warps) {
            const int e = e0 + lane * warps;
            unsigned gaps = __ballot_sync(0xffffffffu, e < p.keys && begin[e] + total[e] < begin[e + 1]);
            for (; gaps; gaps &= gaps - 1) {
                const int g = e0 + (__ffs(gaps) - 1) * warps;
                for (int s = begin[g] + total[g] + lane; s < begin[g + 1]; s += 32) source[s] = -1;
            }
        }
        for (int64_t s = begin[p.keys] + (int64_t)blockIdx.x * SORT_THREADS + threadIdx.x; s < slots; s += (int64_t)gridDim.x * SORT_THREADS) source[s] = -1;
    }
};

// ---- rows to their places ------------------------------------------------------------------------------------------------
#define EXPERT_THREADS 256
#define EXPERT_ZEROS 8  // places that a group looks at for rows of zeros
#define COMBINE_THREADS 128

// A row is n units U of memory: 16 bytes, or an element where rows do not start on 16-byte boundaries.  L lanes take CH units each of a row's tile.
template <typename U, int L, int CH>
__global__ void __launch_bounds__(EXPERT_THREADS)
k_dispatch(const U* x, int64_t x_stride, int64_t rows, int n, int tiles, int k, const int* position, const int* source, U* __restrict__ out, int64_t out_stride,
           int64_t slots) {
    int64_t unit = (int64_t)blockIdx.x * (EXPERT_THREADS / L) + threadIdx.x / L;
    const int t = threadIdx.x % L;
    op_next_may_start();
    op_wait_for_previous();
    const int64_t row = unit / tiles;
    const int first = (int)(unit - row * tiles) * (L * CH) + t;
    if (row < rows) {
        U v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (first + c * L < n) v[c] = x[row * x_stride + first + c * L];
        for (int j = 0; j < k; ++j) {
            const int at = position[row * k + j];
            if ((unsigned)at >= slots) continue;
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (first + c * L < n) out[at * out_stride + first + c * L] = v[c];
        }
        return;
    }
    const int64_t from = (row - rows) * EXPERT_ZEROS, to = min(from + EXPERT_ZEROS, slots);
    for (int64_t s = from; s < to; ++s) {
        if ((unsigned)source[s] < (uint64_t)rows * k) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (first + c * L < n) out[s * out_stride + first + c * L] = U();
    }
}

// J choices' rows are on their way together: of one or two choices with four accesses a lane, of more four with two (30011 x 1000 fp16, k = 8: 88 us; two with four accesses 92, eight with two
// 92; 65536 x 1536 bf16, k = 2: 113 and 118).  Blocks of four warps: of eight 95 us, the former.
template <typename T, int VEC, int L, int CH, int J>
__global__ void __launch_bounds__(COMBINE_THREADS)
k_combine(const T* y, int64_t y_stride, int64_t slots, int64_t rows, int n, int tiles, int k, const int* position, const float* gate, T* __restrict__ out,
          int64_t out_stride) {
    const int64_t unit = (int64_t)blockIdx.x * (COMBINE_THREADS / L) + threadIdx.x / L, row = unit / tiles;
    const int t = threadIdx.x % L, first = ((int)(unit - row * tiles) * (L * CH) + t) * VEC;
    op_next_may_start();
    op_wait_for_previous();
    if (row >= rows) return;
    float acc[CH][VEC];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += J) {
        OpRaw<T, VEC> v[J][CH];
        int at[J];
        float g[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            at[j] = j0 + j < k ? position[row * k + j0 + j] : -1;
            if ((unsigned)at[j] >= slots) at[j] = -1;
            g[j] = at[j] < 0 ? 0.0f : gate ? gate[row * k + j0 + j] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = first + c * L * VEC;
                v[j][c].zero();
                if (at[j] >= 0 && col < n) v[j][c].load(y + at[j] * y_stride + col);
            }
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] = fmaf(g[j], v[j][c].get(i), acc[c][i]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = first + c * L * VEC;
        if (col < n) op_store<T, VEC>(out + row * out_stride + col, acc[c]);
    }
}

// W warps (W = 1: L lanes) walk along a row; K >= k choices at once.
template <typename T, int VEC, int W, int L, int K>
__global__ void __launch_bounds__(EXPERT_THREADS)
k_combine_backward(const T* dout, int64_t dout_stride, const T* y, int64_t y_stride, int64_t slots, int64_t rows, int n, int k, const int* position,
                   const int* source, const float* gate, T* __restrict__ dy, int64_t dy_stride, float* __restrict__ dgate, int64_t row_blocks) {
    constexpr int LANES = W == 1 ? L : 32 * W, PER = EXPERT_THREADS / LANES;
    static_assert(W == 1 || 32 * W == EXPERT_THREADS, "a block per row");
    __shared__ float s_dot[K][W];
    const int t = threadIdx.x % LANES, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    op_next_may_start();
    op_wait_for_previous();
    if ((int64_t)blockIdx.x >= row_blocks) {  // rows of zeros
        const int64_t from = ((int64_t)blockIdx.x - row_blocks) * 32;
        for (int64_t s = from + warp; s < min(from + 32, slots); s += EXPERT_THREADS / 32) {
            if ((unsigned)source[s] < (uint64_t)rows * k) continue;
            float none[VEC] = {};
            for (int64_t col = lane * VEC; col < n; col += 32 * VEC) op_store<T, VEC>(dy + s * dy_stride + col, none);
        }
        return;
    }
    const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    if (L == 32 && row >= rows) return;
    int at[K];
    float g[K], dot[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        at[j] = j < k && row < rows ? position[row * k + j] : -1;
        if ((unsigned)at[j] >= slots) at[j] = -1;
        g[j] = at[j] >= 0 ? gate[row * k + j] : 0.0f;
        dot[j] = 0.0f;
    }
    if (row < rows)
        for (int64_t col = (int64_t)t * VEC; col < n; col += LANES * VEC) {
            OpRaw<T, VEC> d, v[K];
            d.load(dout + row * dout_stride + col);
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (at[j] >= 0) v[j].load(y + at[j] * y_stride + col);
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (at[j] >= 0) {
                    float o[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        dot[j] = fmaf(d.get(i), v[j].get(i), dot[j]);
                        o[i] = g[j] * d.get(i);
                    }
                    op_store<T, VEC>(dy + at[j] * dy_stride + col, o);
                }
        }
#pragma unroll
    for (int j = 0; j < K; ++j) dot[j] = op_group_sum<L>(dot[j]);
    if (W > 1) {
        if (lane == 0)
#pragma unroll
            for (int j = 0; j < K; ++j) s_dot[j][warp] = dot[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < K; ++j) {
            dot[j] = s_dot[j][0];
#pragma unroll
            for (int w = 1; w < W; ++w) dot[j] += s_dot[j][w];
        }
    }
    if (t == 0 && row < rows)
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (j < k) dgate[row * k + j] = at[j] >= 0 ? dot[j] : 0.0f;
}

// ---- which kernel --------------------------------------------------------------------------------------------------------
// f(lanes, units per lane) by a row's units: 8 or 16 lanes up to as many of them, then a warp with one to MOST each; longer rows are tiles.  Single elements are up to eight a lane, or too
// few bytes are on their way (2386 columns of fp16: 59 us with two, 42 so).
template <int MOST, typename F>
void expert_with_shape(int units, F&& f) {
    using std::integral_constant;
    if (units <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (units <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (units <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (units <= 64 || MOST == 2) f(integral_constant<int, 32>(), integral_constant<int, 2>());
    else if (units <= 128 || MOST == 4) f(integral_constant<int, 32>(), integral_constant<int, 4>());
    else f(integral_constant<int, 32>(), integral_constant<int, MOST>());
}
bool expert_blocks(int64_t units, int lanes, int threads, unsigned* blocks) {
    const int64_t b = (units + threads / lanes - 1) / (threads / lanes);
    *blocks = (unsigned)b;
    return b <= INT32_MAX;
}
bool expert_aligned(const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0; }

struct Experts {
    cudaStream_t s;
    int64_t rows, slots;
    int n, k;
    const int *position, *source;
};
template <typename U>
bool dispatch_go(const Experts& a, const void* x, int64_t xs, void* out, int64_t os, int per) {
    const int n = a.n / per;
    bool fits = true;
    expert_with_shape<(sizeof(U) < 16 ? 8 : 4)>(n, [&](auto l, auto ch) {
        constexpr int L = decltype(l)::value, CH = decltype(ch)::value;
        const int tiles = (int)ceil_div64(n, L * CH);
        unsigned blocks;
        fits = expert_blocks((a.rows + (a.slots + EXPERT_ZEROS - 1) / EXPERT_ZEROS) * tiles, L, EXPERT_THREADS, &blocks);
        if (fits)
            op_launch_next(a.s, dim3(blocks), dim3(EXPERT_THREADS), 0, k_dispatch<U, L, CH>, (const U*)x, xs / per, a.rows, n, tiles, a.k, a.position, a.source, (U*)out, os / per, a.slots);
    });
    return fits;
}
template <typename T, int VEC, int J>
bool combine_go(const Experts& a, const void* y, int64_t ys, const float* gate, void* out, int64_t os) {
    bool fits = true;
    expert_with_shape<(VEC == 1 ? 8 : J == 4 ? 2 : 4)>((int)ceil_div64(a.n, VEC), [&](auto l, auto ch) {
        constexpr int L = decltype(l)::value, CH = decltype(ch)::value;
        const int tiles = (int)ceil_div64(a.n, L * CH * VEC);
        unsigned blocks;
        fits = expert_blocks(a.rows * tiles, L, COMBINE_THREADS, &blocks);
        if (fits) op_launch_next(a.s, dim3(blocks), dim3(COMBINE_THREADS), 0, k_combine<T, VEC, L, CH, J>, (const T*)y, ys, a.slots, a.rows, a.n, tiles, a.k, a.position, gate, (T*)out, os);
    });
    return fits;
}
template <typename T, int VEC>
bool combine_pick(const Experts& a, const void* y, int64_t ys, const float* gate, void* out, int64_t os) {
    return a.k == 1 ? combine_go<T, VEC, 1>(a, y, ys, gate, out, os) : a.k == 2 ? combine_go<T, VEC, 2>(a, y, ys, gate, out, os) : combine_go<T, VEC, 4>(a, y, ys, gate, out, os);
}
template <typename T, int VEC, int W, int L>
void combine_backward_go(const Experts& a, const void* dout, int64_t ds, const void* y, int64_t ys, const float* gate, void* dy, int64_t dys, float* dgate) {
    constexpr int PER = EXPERT_THREADS / (W == 1 ? L : 32 * W);
    const int64_t row_blocks = (a.rows + PER - 1) / PER, blocks = row_blocks + (a.slots + 31) / 32;  // below 2^28 + 2^26: eight rows to a block or more, but where rows are few
#define GO(K) \
    op_launch_next(a.s, dim3((unsigned)blocks), dim3(EXPERT_THREADS), 0, k_combine_backward<T, VEC, W, L, K>, (const T*)dout, ds, (const T*)y, ys, a.slots, a.rows, a.n, a.k, a.position, a.source, gate, \
                   (T*)dy, dys, dgate, row_blocks)
    if (a.k <= 1) GO(1);
    else if (a.k <= 2) GO(2);
    else if (a.k <= 4) GO(4);
    else if (a.k <= 8) GO(8);
    else GO(16);
#undef GO
}
template <typename T, int VEC>
void combine_backward_pick(const Experts& a, const void* dout, int64_t ds, const void* y, int64_t ys, const float* gate, void* dy, int64_t dys, float* dgate) {
    // eight lanes for short rows: fewer of them for a sum over the lanes (55049 x 59 bf16, k = 5: 52 us, with a warp per row 60)
    if (a.n <= 8 * VEC || (VEC == 1 && a.n <= 64)) combine_backward_go<T, VEC, 1, 8>(a, dout, ds, y, ys, gate, dy, dys, dgate);
    else if (a.n <= 64 * VEC || a.rows >= 8 * (int64_t)sm_count()) combine_backward_go<T, VEC, 1, 32>(a, dout, ds, y, ys, gate, dy, dys, dgate);
    else combine_backward_go<T, VEC, 8, 32>(a, dout, ds, y, ys, gate, dy, dys, dgate);
}

int expert_check(const Experts& a, int type, char* err, size_t err_len) {
    if (!op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (a.k < 1 || a.k > EXPERT_MAX_K) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "k must be in [1, %d] (got %d)", EXPERT_MAX_K, a.k);
    if (a.rows < 0 || a.rows > INT32_MAX || a.rows * a.k > OP_MAX_ENTRIES || a.slots < 0 || a.slots > OP_MAX_ENTRIES)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows and slots must not be negative, rows * k and slots at most 2^31 - 1024");
    if (a.n < 1 || a.n > OP_MAX_COLUMNS) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "n must be in [1, 2^30] (got %d)", a.n);
    if (a.rows > 0 && !a.position) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_position is NULL");
    if (((uintptr_t)a.position | (uintptr_t)a.source) & 3) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    return TB_OK;
}
int expert_tensor(const OpRows& t, int64_t stride, int n, int size, const char* name, char* err, size_t err_len) {
    if (t.rows == 0) return TB_OK;
    if (!t.p) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    if (t.rows > 1 && stride < n) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "row strides must be at least n");
    if ((uintptr_t)t.p % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    return TB_OK;
}
int expert_too_many(char* err, size_t err_len) { return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows times columns are too many for one launch"); }

}  // namespace

extern "C" int64_t tb_expert_slots(int64_t rows, int k, int experts, int align) {
    if (rows < 0 || rows > INT32_MAX || k < 1 || k > EXPERT_MAX_K || experts < 1 || experts > SORT_MAX_E || align < 1) return TB_ERR_INVALID_ARGUMENT;
    const int64_t entries = rows * k, most = entries + (entries < experts ? entries : experts) * (int64_t)(align - 1);
    return most > OP_MAX_ENTRIES ? TB_ERR_INVALID_ARGUMENT : most / align * align;
}
extern "C" int64_t tb_expert_order_workspace(int64_t rows, int k, int experts) {
    if (tb_expert_slots(rows, k, experts, 1) < 0) return TB_ERR_INVALID_ARGUMENT;
    // for any align: more blocks fill the places that are left over where those are many
    const int64_t usual = sort_words(sort_plan(rows * k, experts, 1)), filling = sort_words(sort_plan(rows * k, experts, 1, INT32_MAX));
    return (usual > filling ? usual : filling) * 4;
}

extern "C" int tb_expert_order(const int32_t* d_index, int64_t rows, int k, int experts, int align, int32_t* d_position, int32_t* d_source, int64_t slots, int32_t* d_offsets, void* d_work,
                               int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    if (experts < 1 || experts > SORT_MAX_E) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "experts must be in [1, %d] (got %d)", SORT_MAX_E, experts);
    if (k < 1 || k > EXPERT_MAX_K) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "k must be in [1, %d] (got %d)", EXPERT_MAX_K, k);
    if (align < 1) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "align must be positive (got %d)", align);
    const int64_t want = tb_expert_slots(rows, k, experts, align);
    if (want < 0) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must not be negative, and rows * k and the places at most 2^31 - 1024");
    if (slots != want) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "slots must be %lld (got %lld)", (long long)want, (long long)slots);
    if (!d_offsets || (rows > 0 && (!d_index || !d_position || !d_source))) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (((uintptr_t)d_index | (uintptr_t)d_position | (uintptr_t)d_source | (uintptr_t)d_offsets) & 3) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const int64_t need = tb_expert_order_workspace(rows, k, experts);
    if (need > 0 && (!d_work || work_bytes < need || ((uintptr_t)d_work & 3)))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    const OpRows ix = op_vector(d_index, rows * k), po = op_vector(d_position, rows * k), so = op_vector(d_source, slots), of = op_vector(d_offsets, experts + 1);
    if (op_meets(ix, {po, so, of}) || op_meets(po, {so, of}) || op_meets(so, {of})) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const SortPlan plan = sort_plan(rows * k, experts, align, slots - rows * k);
    sort_count(s, plan, ExpertSource{d_index}, rows * k, static_cast<int*>(d_work));
    sort_place(s, plan, ExpertSource{d_index}, rows * k, static_cast<int*>(d_work), ExpertPut{d_position, d_source, d_offsets, slots});
    return op_launched(err, err_len);
}

extern "C" int tb_dispatch_forward(const void* d_x, int64_t x_stride, int type, int64_t rows, int n, int k, const int32_t* d_position, const int32_t* d_source, int64_t slots, void* d_out,
                                   int64_t out_stride, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const Experts a = {static_cast<cudaStream_t>(stream), rows, slots, n, k, d_position, d_source};
    int rc = expert_check(a, type, err, err_len);
    if (rc != TB_OK) return rc;
    const int size = op_type_size(type);
    const OpRows xr = {d_x, x_stride * size, rows, (int64_t)n * size}, outr = {d_out, out_stride * size, slots, (int64_t)n * size};
    if ((rc = expert_tensor(xr, x_stride, n, size, "d_x", err, err_len)) != TB_OK || (rc = expert_tensor(outr, out_stride, n, size, "d_out", err, err_len)) != TB_OK) return rc;
    if (slots == 0) return TB_OK;
    if (!d_source) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_source is NULL");
    if (op_extents_meet(outr, {xr, op_vector(d_position, rows * k), op_vector(d_source, slots)})) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_out overlaps another tensor");
    const int per = 16 / size;
    const bool wide = n % per == 0 && expert_aligned(d_x, x_stride, size) && expert_aligned(d_out, out_stride, size);
    const bool fits = wide ? dispatch_go<uint4>(a, d_x, x_stride, d_out, out_stride, per) : size == 4 ? dispatch_go<unsigned>(a, d_x, x_stride, d_out, out_stride, 1)
                                                                                                     : dispatch_go<unsigned short>(a, d_x, x_stride, d_out, out_stride, 1);
    return fits ? op_launched(err, err_len) : expert_too_many(err, err_len);
}

extern "C" int tb_combine_forward(const void* d_y, int64_t y_stride, int type, int64_t slots, int64_t rows, int n, int k, const int32_t* d_position, const float* d_gate, void* d_out, int64_t out_stride,
                                  void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const Experts a = {static_cast<cudaStream_t>(stream), rows, slots, n, k, d_position, nullptr};
    int rc = expert_check(a, type, err, err_len);
    if (rc != TB_OK) return rc;
    const int size = op_type_size(type);
    const OpRows yr = {d_y, y_stride * size, slots, (int64_t)n * size}, outr = {d_out, out_stride * size, rows, (int64_t)n * size};
    if ((rc = expert_tensor(yr, y_stride, n, size, "d_y", err, err_len)) != TB_OK || (rc = expert_tensor(outr, out_stride, n, size, "d_out", err, err_len)) != TB_OK) return rc;
    if ((uintptr_t)d_gate & 3) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    if (rows == 0) return TB_OK;
    if (op_extents_meet(outr, {yr, op_vector(d_position, rows * k), op_vector(d_gate, rows * k)})) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_out overlaps another tensor");
    const bool wide = n % (16 / size) == 0 && expert_aligned(d_y, y_stride, size) && expert_aligned(d_out, out_stride, size);
#define GO(T, VEC) (wide ? combine_pick<T, VEC>(a, d_y, y_stride, d_gate, d_out, out_stride) : combine_pick<T, 1>(a, d_y, y_stride, d_gate, d_out, out_stride))
    const bool fits = type == TB_TYPE_F32 ? GO(float, 4) : type == TB_TYPE_F16 ? GO(__half, 8) : GO(__nv_bfloat16, 8);
#undef GO
    return fits ? op_launched(err, err_len) : expert_too_many(err, err_len);
}

extern "C" int tb_combine_backward(const void* d_dout, int64_t dout_stride, const void* d_y, int64_t y_stride, int type, int64_t slots, int64_t rows, int n, int k, const int32_t* d_position,
                                   const int32_t* d_source, const float* d_gate, void* d_dy, int64_t dy_stride, float* d_dgate, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const Experts a = {static_cast<cudaStream_t>(stream), rows, slots, n, k, d_position, d_source};
    int rc = expert_check(a, type, err, err_len);
    if (rc != TB_OK) return rc;
    const int size = op_type_size(type);
    const int64_t row = (int64_t)n * size;
    const OpRows gr = {d_dout, dout_stride * size, rows, row}, yr = {d_y, y_stride * size, slots, row}, dr = {d_dy, dy_stride * size, slots, row};
    if ((rc = expert_tensor(gr, dout_stride, n, size, "d_dout", err, err_len)) != TB_OK || (rc = expert_tensor(yr, y_stride, n, size, "d_y", err, err_len)) != TB_OK ||
        (rc = expert_tensor(dr, dy_stride, n, size, "d_dy", err, err_len)) != TB_OK)
        return rc;
    if ((rows > 0 && (!d_gate || !d_dgate)) || (slots > 0 && !d_source)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (((uintptr_t)d_gate | (uintptr_t)d_dgate) & 3) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    const OpRows po = op_vector(d_position, rows * k), so = op_vector(d_source, slots), ga = op_vector(d_gate, rows * k), dg = op_vector(d_dgate, rows * k);
    if (op_extents_meet(dr, {gr, yr, po, so, ga, dg}) || op_extents_meet(dg, {gr, yr, po, so, ga})) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    if (rows == 0 && slots == 0) return TB_OK;
    const bool wide = n % (16 / size) == 0 && expert_aligned(d_dout, dout_stride, size) && expert_aligned(d_y, y_stride, size) && expert_aligned(d_dy, dy_stride, size);
#define GO(T, VEC) (wide ? combine_backward_pick<T, VEC>(a, d_dout, dout_stride, d_y, y_stride, d_gate, d_dy, dy_stride, d_dgate) : combine_backward_pick<T, 1>(a, d_dout, dout_stride, d_y, y_stride, d_gate, d_dy, dy_stride, d_dgate))
    if (type == TB_TYPE_F32) GO(float, 4);
    else if (type == TB_TYPE_F16) GO(__half, 8);
    else GO(__nv_bfloat16, 8);
#undef GO
    return op_launched(err, err_len);
}
