// Choice of k of E experts (LayerStack buckets) per row from a row of logits, with the gates, the per-expert counts, a balance loss and
// a z loss, and the gradient of gates and losses with respect to the logits.
//
//   choice     the k largest logits in descending order, ties to the lowest index.  A logit of -inf forbids its expert; a row whose mask
//              byte is 0, or with nothing but -inf, is empty: index -1, gate 0, not counted
//   p          softmax(l) over the row; gate_j = exp(l_cj) / sum over the chosen (renormalise), else p_cj
//   N, c_e     rows that are not empty, and how often expert e was chosen;  P_e = sum of p_e over the rows / N
//   losses     balance = E * sum_e c_e / (N k) * P_e (the counts are constants to the gradient),  z = sum lse^2 / N
//   backward   h_e = dB E c_e / (N k) / N,  dl = p (h - sum(p h)) + dZ 2 lse / N p + the gates' part: renormalised
//              g_j (dg_j - sum(g dg)) at the chosen, else p_cj dg_j at the chosen - p sum(g dg)
//
// A group of G lanes owns a row and keeps it in registers, V logits per lane; every logit is read once.  The choice compares order-preserving
// integer keys of the logits as they are, so it does not depend on how the softmax rounds.  Bound by memory for wide rows of
// many experts and by latency for the handful of experts of a net.  Sums: fp32 chains over a group's rows, then the groups of a
// block in order, then the blocks in order in 64 bits (second kernel): results repeat bit for bit.
#include "op_common.cuh"

#include <float.h>

namespace {

#define ROUTE_THREADS 512
#define ROUTE_MAX_K 16
#define ROUTE_MAX_E 1024
#define KEY_NEG_INF 0x007fffffu

// unsigned keys in the order of the floats; both zeros alike; a NaN is larger than any number
__device__ __forceinline__ unsigned route_key(float v) {
    if (v != v) return 0xffffffffu;
    const unsigned u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float route_unkey(unsigned k) {
    if (k == 0xffffffffu) return __int_as_float(0x7fc00000);
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

template <int G>
__device__ __forceinline__ unsigned group_max(unsigned v) {
    if (G == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int G>
__device__ __forceinline__ int group_min(int v) {
    if (G == 32) return __reduce_min_sync(0xffffffffu, v);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// the expert of a lane's v-th logit
template <int G, int VEC>
__device__ __forceinline__ int route_expert(int v, int lane) { return (v / VEC) * G * VEC + lane * VEC + v % VEC; }

template <typename T, int G, int V, int VEC>
__device__ __forceinline__ void route_load(const T* row, int experts, int lane, float (&l)[V]) {
#pragma unroll
    for (int c = 0; c < V / VEC; ++c) {
        const int e = c * G * VEC + lane * VEC;
        float t[VEC];
        if (e < experts) {
            op_load<T, VEC>(row + e, t);
#pragma unroll
            for (int i = 0; i < VEC; ++i) l[c * VEC + i] = t[i];
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) l[c * VEC + i] = -INFINITY;
        }
    }
}

// The sums of a launch: counts, rows and probability sums of every block.  part_p [blocks][E] floats, part_c [blocks][E + 1] ints (the last
// is the block's rows), part_z [blocks] floats.
struct RouteParts {
    float* p;
    float* z;
    int* c;
};

template <typename T, int G, int V, int VEC>
__global__ void __launch_bounds__(ROUTE_THREADS)
k_route_forward(const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ mask, int64_t rows, int experts, int k, int renormalise,
                int* __restrict__ index, float* __restrict__ gate, RouteParts part) {
    constexpr int GROUPS = ROUTE_THREADS / G, SLOTS = ROUTE_MAX_K > G ? ROUTE_MAX_K / G : 1;
    extern __shared__ int s_dyn[];
    int* s_count = s_dyn;                                       // [experts + 1]
    float* s_p = reinterpret_cast<float*>(s_dyn + experts + 1);  // [16 warps][experts]
    __shared__ float s_z[ROUTE_THREADS / 32];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, wl = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= experts; e += ROUTE_THREADS) s_count[e] = 0;
    __syncthreads();
    float sum_p[V], sum_z = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum_p[v] = 0.0f;
    int n_rows = 0;
    // every lane of a warp takes the same number of turns: the group reductions want whole warps
    const int64_t first = (int64_t)blockIdx.x * GROUPS + (threadIdx.x / 32) * (32 / G);
    for (int64_t base = first; base < rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = base + group % (32 / G);
        const bool exists = row < rows;
        const bool in = exists && (!mask || mask[row]);
        float l[V];
        if (in) {
            route_load<T, G, V, VEC>(logits + row * stride, experts, lane, l);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) l[v] = -INFINITY;
        }
        unsigned key[V];
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = route_key(l[v]);
        unsigned top = 0;
        float top_l = 0.0f, chosen_sum = 0.0f, total = 0.0f;
        int mine[SLOTS];
        float mine_g[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            mine[s] = -1;
            mine_g[s] = 0.0f;
        }
        bool live = false;
        for (int j = 0; j < k; ++j) {
            unsigned best = 0;
            int at = INT32_MAX;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (key[v] > best) {
                    best = key[v];
                    at = route_expert<G, VEC>(v, lane);
                }
            const unsigned m = group_max<G>(best);
            if (j == 0) {
                top = m;
                live = m > KEY_NEG_INF;
                top_l = live ? route_unkey(top) : 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    l[v] = live ? expf(l[v] - top_l) : 0.0f;
                    total += l[v];
                }
                total = op_group_sum<G>(total);
            }
            const bool ok = m > KEY_NEG_INF;
            const int e = group_min<G>(best == m ? at : INT32_MAX);
            const float g = ok ? expf(route_unkey(m) - top_l) : 0.0f;
            chosen_sum += g;
            if (ok) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (route_expert<G, VEC>(v, lane) == e) key[v] = 0;
            }
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
                if (ok && j == s * G + lane) {
                    mine[s] = e;
                    mine_g[s] = g;
                }
        }
        const float norm = renormalise ? chosen_sum : total;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int j = s * G + lane;
            if (exists && j < k) {
                index[row * k + j] = mine[s];
                gate[row * k + j] = mine[s] >= 0 ? mine_g[s] / norm : 0.0f;
                if (mine[s] >= 0) atomicAdd(&s_count[mine[s]], 1);
            }
        }
        if (live) {
            const float inv = 1.0f / total;
#pragma unroll
            for (int v = 0; v < V; ++v) sum_p[v] = fmaf(l[v], inv, sum_p[v]);
            if (lane == 0) {
                const float lse = top_l + logf(total);
                sum_z = fmaf(lse, lse, sum_z);
                ++n_rows;
            }
        }
    }
    if (n_rows) atomicAdd(&s_count[experts], n_rows);
    // the groups of a warp in halves, then the warps in order
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float t = sum_p[v];
#pragma unroll
        for (int o = 16; o >= G; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        const int e = route_expert<G, VEC>(v, lane);
        if (wl < G && e < experts) s_p[warp * experts + e] = t;
    }
    sum_z = op_group_sum<32>(sum_z);
    if (wl == 0) s_z[warp] = sum_z;
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += ROUTE_THREADS) {
        part.c[(int64_t)blockIdx.x * (experts + 1) + e] = s_count[e];
        if (e < experts) {
            float t = s_p[e];
#pragma unroll
            for (int w = 1; w < ROUTE_THREADS / 32; ++w) t += s_p[w * experts + e];
            part.p[(int64_t)blockIdx.x * experts + e] = t;
        }
    }
    if (threadIdx.x == 0) {
        float t = s_z[0];
        for (int w = 1; w < ROUTE_THREADS / 32; ++w) t += s_z[w];
        part.z[blockIdx.x] = t;
    }
}

// The blocks' sums: one block; S = 1024 / width threads per expert add every S-th block, then those in order, in 64 bits.
__global__ void __launch_bounds__(1024) k_route_final(RouteParts part, int blocks, int experts, int width, int k, int* __restrict__ counts,
                                                       int* __restrict__ rows_out, float* __restrict__ prob_mean, float* __restrict__ losses) {
    __shared__ double s_p[1024];
    __shared__ int s_c[1024];
    __shared__ int s_rows;
    const int e = threadIdx.x % width, slice = threadIdx.x / width, slices = 1024 / width;
    double p = 0.0, z = 0.0;
    int c = 0, n = 0;
    if (e < experts)
#pragma unroll 4
        for (int b = slice; b < blocks; b += slices) {
            p += (double)part.p[(int64_t)b * experts + e];
            c += part.c[(int64_t)b * (experts + 1) + e];
        }
    s_p[threadIdx.x] = p;
    s_c[threadIdx.x] = c;
    if (threadIdx.x == 0) s_rows = 0;
    __syncthreads();
    if (slice == 0)
        for (int s = 1; s < slices; ++s) {
            p += s_p[s * width + e];
            c += s_c[s * width + e];
        }
    for (int b = threadIdx.x; b < blocks; b += 1024) {
        z += (double)part.z[b];
        n += part.c[(int64_t)b * (experts + 1) + experts];
    }
    if (n) atomicAdd(&s_rows, n);
    __syncthreads();
    const int rows = s_rows;
    const double inv = 1.0 / (double)(rows > 0 ? rows : 1);
    const bool owner = slice == 0 && e < experts;
    if (owner) {
        counts[e] = c;
        prob_mean[e] = (float)(p * inv);
    }
    // both losses by a tree over the threads
    s_p[threadIdx.x] = owner ? p * inv * (double)c : 0.0;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if (threadIdx.x < o) s_p[threadIdx.x] += s_p[threadIdx.x + o];
        __syncthreads();
    }
    const double balance = s_p[0] * (double)experts * inv / (double)k;
    __syncthreads();
    s_p[threadIdx.x] = z;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if (threadIdx.x < o) s_p[threadIdx.x] += s_p[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        losses[0] = (float)balance;
        losses[1] = (float)(s_p[0] * inv);
        *rows_out = rows;
    }
}

template <typename T, int G, int V, int VEC>
__global__ void __launch_bounds__(256)
k_route_backward(const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ mask, int64_t rows, int experts, int k, int renormalise,
                 const int* __restrict__ index, const float* __restrict__ gate, const float* __restrict__ dgate, const int* __restrict__ counts,
                 const int* __restrict__ n_rows, const float* __restrict__ dlosses, T* __restrict__ dlogits, int64_t dstride) {
    constexpr int GROUPS = 256 / G, SLOTS = ROUTE_MAX_K > G ? ROUTE_MAX_K / G : 1;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float n = (float)max(*n_rows, 1);
    const float db = dlosses ? dlosses[0] : 0.0f, dz = dlosses ? dlosses[1] : 0.0f;
    const float hk = db * (float)experts / (n * (float)k) / n, zk = 2.0f * dz / n;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = route_expert<G, VEC>(v, lane);
        h[v] = e < experts ? hk * (float)counts[e] : 0.0f;
    }
    const int64_t first = (int64_t)blockIdx.x * GROUPS + (threadIdx.x / 32) * (32 / G);
    for (int64_t base = first; base < rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = base + group % (32 / G);
        const bool exists = row < rows;
        const bool in = exists && (!mask || mask[row]);
        float l[V];
        if (in) {
            route_load<T, G, V, VEC>(logits + row * stride, experts, lane, l);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) l[v] = -INFINITY;
        }
        int at[SLOTS];
        float ga[SLOTS], dg[SLOTS], dot = 0.0f;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int j = s * G + lane;
            const bool mine = in && j < k;
            at[s] = mine ? index[row * k + j] : -1;
            const bool ok = at[s] >= 0;
            ga[s] = ok ? gate[row * k + j] : 0.0f;
            dg[s] = ok && dgate ? dgate[row * k + j] : 0.0f;
            dot = fmaf(ga[s], dg[s], dot);
        }
        dot = op_group_sum<G>(dot);
        unsigned best = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) best = max(best, route_key(l[v]));
        best = group_max<G>(best);
        const bool live = best > KEY_NEG_INF;
        const float top_l = live ? route_unkey(best) : 0.0f;
        float total = 0.0f, ph = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] = live ? expf(l[v] - top_l) : 0.0f;
            total += l[v];
            ph = fmaf(l[v], h[v], ph);
        }
        total = op_group_sum<G>(total);
        total = live ? total : 1.0f;
        ph = op_group_sum<G>(ph) / total;
        const float shift = zk * (top_l + logf(total)) - ph - (renormalise ? 0.0f : dot), inv = 1.0f / total;
#pragma unroll
        for (int v = 0; v < V; ++v) l[v] = l[v] * inv * (h[v] + shift);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const float add = ga[s] * (renormalise ? dg[s] - dot : dg[s]);
            for (int j = 0; j < G && s * G + j < k; ++j) {
                const int e = __shfl_sync(0xffffffffu, at[s], j, G);
                const float a = __shfl_sync(0xffffffffu, add, j, G);
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (route_expert<G, VEC>(v, lane) == e) l[v] += a;
            }
        }
        if (!exists) continue;
        T* out = dlogits + row * dstride;
#pragma unroll
        for (int c = 0; c < V / VEC; ++c) {
            const int e = c * G * VEC + lane * VEC;
            if (e < experts) {
                float t[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) t[i] = live ? l[c * VEC + i] : 0.0f;
                op_store<T, VEC>(out + e, t);
            }
        }
    }
}

// Lanes per row and logits per lane by the number of experts: groups as small as eight logits a lane allow, so that few lanes idle and the
// reductions are short; whole warps from 129 experts on.
#define ROUTE_SHAPES(GO) \
    if (experts <= 16) { GO(4, 4); } else if (experts <= 64) { GO(8, 8); } else if (experts <= 128) { GO(16, 8); } \
    else if (experts <= 256) { GO(32, 8); } else if (experts <= 512) { GO(32, 16); } else { GO(32, 32); }

int route_group(int experts) { return experts <= 16 ? 4 : experts <= 64 ? 8 : experts <= 128 ? 16 : 32; }
int route_forward_blocks(int64_t rows, int experts) {
    const int64_t groups = ROUTE_THREADS / route_group(experts), want = (rows + groups - 1) / groups, most = 2 * (int64_t)sm_count();
    return (int)(want < 1 ? 1 : want < most ? want : most);
}
size_t route_smem(int experts) { return (size_t)(experts + 1 + ROUTE_THREADS / 32 * experts) * 4; }

template <typename T>
void route_forward_go(cudaStream_t s, const void* logits, int64_t stride, const uint8_t* mask, int64_t rows, int experts, int k, int renormalise, int* index,
                      float* gate, RouteParts part, bool wide) {
    constexpr int W = 16 / (int)sizeof(T);
    const int blocks = route_forward_blocks(rows, experts);
    const size_t smem = route_smem(experts);
#define GO(G, V)                                                                                                                                \
    do {                                                                                                                                        \
        constexpr int VW = W < (V) ? W : (V);                                                                                                   \
        auto kern = wide ? k_route_forward<T, G, V, VW> : k_route_forward<T, G, V, 1>;                                                          \
        if (smem > 40000) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);                                   \
        kern<<<blocks, ROUTE_THREADS, smem, s>>>((const T*)logits, stride, mask, rows, experts, k, renormalise, index, gate, part);             \
    } while (0)
    ROUTE_SHAPES(GO)
#undef GO
}
template <typename T>
void route_backward_go(cudaStream_t s, const void* logits, int64_t stride, const uint8_t* mask, int64_t rows, int experts, int k, int renormalise,
                       const int* index, const float* gate, const float* dgate, const int* counts, const int* n_rows, const float* dlosses, void* dlogits,
                       int64_t dstride, bool wide) {
    constexpr int W = 16 / (int)sizeof(T);
    const int64_t groups = 256 / route_group(experts), want = (rows + groups - 1) / groups, most = 8 * (int64_t)sm_count();
    const int blocks = (int)(want < most ? want : most);
#define GO(G, V)                                                                                                                              \
    do {                                                                                                                                      \
        constexpr int VW = W < (V) ? W : (V);                                                                                                 \
        auto kern = wide ? k_route_backward<T, G, V, VW> : k_route_backward<T, G, V, 1>;                                                      \
        kern<<<blocks, 256, 0, s>>>((const T*)logits, stride, mask, rows, experts, k, renormalise, index, gate, dgate, counts, n_rows, dlosses, \
                                    (T*)dlogits, dstride);                                                                                    \
    } while (0)
    ROUTE_SHAPES(GO)
#undef GO
}

bool route_wide(const void* p, int64_t stride, int experts, int size) {
    const int bytes = experts <= 16 && size == 2 ? 8 : 16;  // four logits a lane
    return (uintptr_t)p % bytes == 0 && (stride * size) % bytes == 0 && ((int64_t)experts * size) % bytes == 0;
}

int route_check(int type, int64_t rows, int experts, int k, const void* logits, int64_t stride, char* err, size_t err_len) {
    const int size = op_type_size(type);
    if (!size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "type must be TB_TYPE_F32, TB_TYPE_F16 or TB_TYPE_BF16 (got %d)", type);
    if (experts < 1 || experts > ROUTE_MAX_E) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "experts must be in [1, %d] (got %d)", ROUTE_MAX_E, experts);
    if (k < 1 || k > experts || k > ROUTE_MAX_K) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "k must be in [1, min(experts, %d)] (got %d)", ROUTE_MAX_K, k);
    if (rows < 0 || rows * k > INT32_MAX) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must not be negative and rows * k below 2^31");
    if (rows > 0 && !logits) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_logits is NULL");
    if (rows > 1 && stride < experts) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the row stride must be at least experts");
    if ((uintptr_t)logits % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_logits must be aligned to its elements");
    return TB_OK;
}

}  // namespace

extern "C" int64_t tb_route_forward_workspace(int64_t rows, int experts) {
    if (rows < 0 || experts < 1 || experts > ROUTE_MAX_E) return TB_ERR_INVALID_ARGUMENT;
    return (int64_t)route_forward_blocks(rows, experts) * (2 * experts + 2) * 4;
}

extern "C" int tb_route_forward(const void* d_logits, int64_t stride, int type, int64_t rows, int experts, int k, int renormalise, const uint8_t* d_mask,
                                int32_t* d_index, float* d_gate, int32_t* d_counts, int32_t* d_rows, float* d_prob_mean, float* d_losses, void* d_work,
                                int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int rc = route_check(type, rows, experts, k, d_logits, stride, err, err_len);
    if (rc != TB_OK) return rc;
    if ((rows > 0 && (!d_index || !d_gate)) || !d_counts || !d_rows || !d_prob_mean || !d_losses)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "an output pointer is NULL");
    const int64_t need = tb_route_forward_workspace(rows, experts);
    if (!d_work || work_bytes < need || ((uintptr_t)d_work & 3))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int blocks = route_forward_blocks(rows, experts);
    RouteParts part;
    part.p = static_cast<float*>(d_work);
    part.c = reinterpret_cast<int*>(part.p + (size_t)blocks * experts);
    part.z = reinterpret_cast<float*>(part.c + (size_t)blocks * (experts + 1));
    const bool wide = route_wide(d_logits, stride, experts, op_type_size(type));
#define ARGS s, d_logits, stride, d_mask, rows, experts, k, renormalise, d_index, d_gate, part, wide
    if (type == TB_TYPE_F32) route_forward_go<float>(ARGS);
    else if (type == TB_TYPE_F16) route_forward_go<__half>(ARGS);
    else route_forward_go<__nv_bfloat16>(ARGS);
#undef ARGS
    int width = 1;
    while (width < experts) width *= 2;
    k_route_final<<<1, 1024, 0, s>>>(part, blocks, experts, width, k, d_counts, d_rows, d_prob_mean, d_losses);
    return op_launched(err, err_len);
}

extern "C" int tb_route_backward(const void* d_logits, int64_t stride, int type, int64_t rows, int experts, int k, int renormalise, const uint8_t* d_mask,
                                 const int32_t* d_index, const float* d_gate, const float* d_dgate, const int32_t* d_counts, const int32_t* d_rows,
                                 const float* d_dlosses, void* d_dlogits, int64_t dstride, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int rc = route_check(type, rows, experts, k, d_logits, stride, err, err_len);
    if (rc != TB_OK) return rc;
    if (rows == 0) return TB_OK;
    if (!d_index || !d_gate || !d_counts || !d_rows || !d_dlogits) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a device pointer is NULL");
    if (rows > 1 && dstride < experts) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the row stride must be at least experts");
    if ((uintptr_t)d_dlogits % op_type_size(type)) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dlogits must be aligned to its elements");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = route_wide(d_logits, stride, experts, op_type_size(type)) && route_wide(d_dlogits, dstride, experts, op_type_size(type));
#define ARGS s, d_logits, stride, d_mask, rows, experts, k, renormalise, d_index, d_gate, d_dgate, d_counts, d_rows, d_dlosses, d_dlogits, dstride, wide
    if (type == TB_TYPE_F32) route_backward_go<float>(ARGS);
    else if (type == TB_TYPE_F16) route_backward_go<__half>(ARGS);
    else route_backward_go<__nv_bfloat16>(ARGS);
#undef ARGS
    return op_launched(err, err_len);
}
