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
// A group of G lanes owns a row and keeps it in registers, V logits per lane; every logit is read once.  The choice compares integer words
// made of the logits' bits as they are and the expert, so it does not depend on how the softmax rounds.  Sums: fp32 chains over a group's
// rows, then the groups of a block in order, then the blocks in order in 64 bits (second kernel): results repeat bit for bit.
//
// What bounds it are issue slots for many experts (490 instructions per row of 256 bf16 logits and eight choices, slots at 73 %: 29 us for 40000
// rows, whose bytes would take 3.5; their gradient 20 us at 290 instructions per row) and latency for the handful of a net (65536 x 9 fp32, one choice:
// 10 us with both launches, the gradient 5.3).
#include "op_common.cuh"

namespace {

#define ROUTE_THREADS 512
#define ROUTE_MAX_K 16
#define ROUTE_MAX_E 1024

// A logit and its expert as one unsigned word that orders like (logit, -expert): the order-preserving key of the logit's bits above the
// expert's complement.  16-bit logits make 32-bit words, 32-bit ones 64-bit words.  Both zeros are alike, a NaN is larger than any number; words are
// distinct, so the k-th largest is one comparison, ties included.
template <typename T> struct RouteWord;
template <> struct RouteWord<float> {
    using W = unsigned long long;
    static constexpr W NONE = ((W)0x007fffffu << 32) | 0xffffffffu;  // of -inf: words above it can be chosen
    template <int N>
    static __device__ __forceinline__ W make(const OpRaw<float, N>& l, int i, int e) {
        const float x = l.get(i);
        const unsigned u = __float_as_uint(x + 0.0f);
        const unsigned key = x != x ? 0xffffffffu : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
        return ((W)key << 32) | (unsigned)~e;
    }
    static __device__ __forceinline__ int expert(W w) { return (int)~(unsigned)w; }
    static __device__ __forceinline__ float logit(W w) {
        const unsigned k = (unsigned)(w >> 32);
        return k == 0xffffffffu ? __int_as_float(0x7fc00000) : __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
    }
    template <int G>
    static __device__ __forceinline__ W group_max(W w) {
        if (G == 32) {
            const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(w >> 32));
            const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(w >> 32) == hi ? (unsigned)w : 0u);
            return ((W)hi << 32) | lo;
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, o));
        return w;
    }
};
template <typename T> struct RoutePair;
template <> struct RoutePair<__half> {
    using P = __half2;
    static __device__ __forceinline__ P zeros() { return __float2half2_rn(0.0f); }
};
template <> struct RoutePair<__nv_bfloat16> {
    using P = __nv_bfloat162;
    static __device__ __forceinline__ P zeros() { return __float2bfloat162_rn(0.0f); }
};
template <typename T, unsigned NEG_INF>
struct RouteWord16 {
    using W = unsigned;
    static constexpr W NONE = (NEG_INF << 16) | 0xffffu;
    // Two logits' keys at once: x + 0 makes both zeros alike and every NaN 0x7fff, whose key is the largest.
    static __device__ __forceinline__ unsigned keys(unsigned pair) {
        using P = typename RoutePair<T>::P;
        const P sum = __hadd2(*reinterpret_cast<const P*>(&pair), RoutePair<T>::zeros());
        const unsigned u = *reinterpret_cast<const unsigned*>(&sum);
        return u ^ ((u >> 15 & 0x00010001u) * 0x7fffu + 0x80008000u);
    }
    template <int N>
    static __device__ __forceinline__ W make(const OpRaw<T, N>& l, int i, int e) {
        const unsigned k = keys(l.w[i / 2]);
        return (i & 1 ? k & 0xffff0000u : k << 16) | (0xffffu - (unsigned)e);
    }
    static __device__ __forceinline__ int expert(W w) { return (int)(0xffffu - (w & 0xffffu)); }
    static __device__ __forceinline__ float logit(W w) {
        const unsigned k = w >> 16;
        const unsigned short u = (unsigned short)(k ^ ((k >> 15) ? 0x8000u : 0xffffu));
        return k == 0xffffu ? __int_as_float(0x7fc00000) : op_float(*reinterpret_cast<const T*>(&u));
    }
    template <int G>
    static __device__ __forceinline__ W group_max(W w) {
        if (G == 32) return __reduce_max_sync(0xffffffffu, w);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, o));
        return w;
    }
};
template <> struct RouteWord<__half> : RouteWord16<__half, 0x03ffu> {};
template <> struct RouteWord<__nv_bfloat16> : RouteWord16<__nv_bfloat16, 0x007fu> {};

// the expert of a lane's v-th logit
template <int G, int VEC>
__device__ __forceinline__ int route_expert(int v, int lane) { return (v / VEC) * G * VEC + lane * VEC + v % VEC; }

// -inf in every element of a register
template <typename T> __device__ __forceinline__ unsigned route_never();
template <> __device__ __forceinline__ unsigned route_never<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned route_never<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ unsigned route_never<__nv_bfloat16>() { return 0xff80ff80u; }

// a lane's logits, -inf where there are none
template <typename T, int G, int V, int VEC>
__device__ __forceinline__ void route_load(const T* row, bool in, int experts, int lane, OpRaw<T, VEC> (&l)[V / VEC]) {
#pragma unroll
    for (int c = 0; c < V / VEC; ++c) {
        const int e = c * G * VEC + lane * VEC;
        if (in && e < experts) {
            l[c].load(row + e);
        } else {
#pragma unroll
            for (int i = 0; i < OpRaw<T, VEC>::WORDS; ++i) l[c].w[i] = route_never<T>();
        }
    }
}

// exp(x - top) of a whole row, as a power of two: the product's rounding costs |x - top| 2^-24 of a probability, so 1e-6 of one of e^-16; exp(-inf) is 0
__device__ __forceinline__ float route_exp(float x, float top) {
    float y = (x - top) * 1.44269504f;
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
    return y;
}

// descending, by Batcher's odd-even merges
template <typename W, int N>
__device__ __forceinline__ void route_sort(W (&w)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (p * 2) == (i + j + k) / (p * 2)) {
                        const W a = w[i + j], b = w[i + j + k];
                        w[i + j] = max(a, b);
                        w[i + j + k] = min(a, b);
                    }
}

// The sums of a launch: counts, rows and probability sums of every block.  p [blocks][E], c [blocks][E + 1] (the last is the block's
// rows), z [blocks]; balance [ceil(E / 32)] and ticket belong to the second kernel.
struct RouteParts {
    double* balance;
    float* p;
    float* z;
    int* c;
    int* ticket;
};

// SORTED: a lane sorts its logits once and gives the largest away in every round, which pays from three choices on (16-bit logits, 256 experts, k = 8:
// 1040 instructions per row when every round looks at all of them).
template <typename T, int G, int V, int VEC, bool SORTED>
__global__ void __launch_bounds__(ROUTE_THREADS)
k_route_forward(const T* __restrict__ logits, int64_t stride, const uint8_t* __restrict__ mask, int64_t rows, int experts, int k, int renormalise,
                int* __restrict__ index, float* __restrict__ gate, RouteParts part) {
    using R = RouteWord<T>;
    using W = typename R::W;
    constexpr int GROUPS = ROUTE_THREADS / G, SLOTS = ROUTE_MAX_K > G ? ROUTE_MAX_K / G : 1;
    extern __shared__ int s_dyn[];
    int* s_count = s_dyn;                                       // [experts + 1]
    float* s_p = reinterpret_cast<float*>(s_dyn + experts + 1);  // [16 warps][experts]
    __shared__ float s_z[ROUTE_THREADS / 32];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, wl = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= experts; e += ROUTE_THREADS) s_count[e] = 0;
    op_next_may_start();
    op_wait_for_previous();
    if (blockIdx.x == 0 && threadIdx.x == 0) *part.ticket = 0;
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
        OpRaw<T, VEC> raw[V / VEC];
        route_load<T, G, V, VEC>(logits + row * stride, in, experts, lane, raw);
        W w[V];
#pragma unroll
        for (int v = 0; v < V; ++v) w[v] = R::make(raw[v / VEC], v % VEC, route_expert<G, VEC>(v, lane));
        if (SORTED) route_sort<W, V>(w);
        W mine[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) mine[s] = 0;
        W top = 0;
        for (int j = 0; j < k; ++j) {
            W best = w[0];
            if (!SORTED)
#pragma unroll
                for (int v = 1; v < V; ++v) best = max(best, w[v]);
            const W m = R::template group_max<G>(best);
            if (j == 0) top = m;
            if (SORTED) {
                if (best == m) {
#pragma unroll
                    for (int v = 0; v + 1 < V; ++v) w[v] = w[v + 1];
                    w[V - 1] = 0;
                }
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (w[v] == m) w[v] = 0;
            }
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
                if (j == s * G + lane) mine[s] = m;
        }
        const bool live = top > R::NONE;
        const float top_l = live ? R::logit(top) : 0.0f;
        float l[V], total = 0.0f, chosen = 0.0f, g[SLOTS];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] = route_exp(raw[v / VEC].get(v % VEC), top_l);  // a row that is not live has nothing but -inf
            total += l[v];
        }
        total = op_group_sum<G>(total);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            g[s] = mine[s] > R::NONE ? expf(R::logit(mine[s]) - top_l) : 0.0f;
            chosen += g[s];
        }
        chosen = op_group_sum<G>(chosen);
        const float norm = renormalise ? chosen : total;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int j = s * G + lane;
            if (exists && j < k) {
                const bool ok = mine[s] > R::NONE;
                const int e = ok ? R::expert(mine[s]) : -1;
                index[row * k + j] = e;
                gate[row * k + j] = ok ? g[s] / norm : 0.0f;
                if (ok) atomicAdd(&s_count[e], 1);
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
#pragma unroll
        for (int w = 1; w < ROUTE_THREADS / 32; ++w) t += s_z[w];
        part.z[blockIdx.x] = t;
    }
}

// The blocks' sums, 32 experts per block of 32 warps: lane l of warp w adds expert l of the blocks w, w + 32, .., then warp l adds those of expert l
// in halves, all in 64 bits.  The last block to finish adds up the balance loss of the others, in order.
__global__ void __launch_bounds__(1024) k_route_final(RouteParts part, int blocks, int experts, int k, int* __restrict__ counts, int* __restrict__ rows_out,
                                                       float* __restrict__ prob_mean, float* __restrict__ losses) {
    __shared__ double s_p[32][33], s_z[32], s_b[32];
    __shared__ int s_c[32][33], s_n[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = blockIdx.x * 32;
    double p = 0.0, z = 0.0;
    int c = 0, n = 0;
    op_next_may_start();
    op_wait_for_previous();
    if (e0 + lane < experts)
#pragma unroll 8
        for (int b = warp; b < blocks; b += 32) {
            p += (double)part.p[(int64_t)b * experts + e0 + lane];
            c += part.c[(int64_t)b * (experts + 1) + e0 + lane];
        }
    for (int b = threadIdx.x; b < blocks; b += 1024) {
        z += (double)part.z[b];
        n += part.c[(int64_t)b * (experts + 1) + experts];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) {
        s_z[warp] = z;
        s_n[warp] = n;
    }
    s_p[warp][lane] = p;
    s_c[warp][lane] = c;
    __syncthreads();
    p = s_p[lane][warp];
    c = __reduce_add_sync(0xffffffffu, s_c[lane][warp]);
    n = __reduce_add_sync(0xffffffffu, s_n[lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) p += __shfl_xor_sync(0xffffffffu, p, o);
    const double inv = 1.0 / (double)(n > 0 ? n : 1);
    if (lane == 0) {
        const bool owner = e0 + warp < experts;
        s_b[warp] = owner ? p * inv * (double)c : 0.0;
        if (owner) {
            counts[e0 + warp] = c;
            prob_mean[e0 + warp] = (float)(p * inv);
        }
    }
    __syncthreads();
    if (warp != 0) return;
    double balance = s_b[lane];
    z = s_z[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        balance += __shfl_xor_sync(0xffffffffu, balance, o);
        z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    if (lane != 0) return;
    if (gridDim.x > 1) {
        part.balance[blockIdx.x] = balance;
        __threadfence();
        if (atomicAdd(part.ticket, 1) != (int)gridDim.x - 1) return;
        __threadfence();
        balance = 0.0;
        for (unsigned b = 0; b < gridDim.x; ++b) balance += *static_cast<volatile double*>(part.balance + b);
    }
    losses[0] = (float)(balance * (double)experts * inv / (double)k);
    losses[1] = (float)(z * inv);
    *rows_out = n;
}

// dlogits may be the logits: a group reads its row before it writes it
template <typename T, int G, int V, int VEC>
__global__ void __launch_bounds__(256)
k_route_backward(const T* logits, int64_t stride, const uint8_t* __restrict__ mask, int64_t rows, int experts, int k, int renormalise,
                 const int* __restrict__ index, const float* __restrict__ gate, const float* __restrict__ dgate, const int* __restrict__ counts,
                 const int* __restrict__ n_rows, const float* __restrict__ dlosses, T* dlogits, int64_t dstride) {
    constexpr int GROUPS = 256 / G, SLOTS = ROUTE_MAX_K > G ? ROUTE_MAX_K / G : 1;
    // the gates' part of a group's row: zero but while the chosen experts' lanes pass it to the lanes that hold those logits
    __shared__ __align__(16) float s_add[GROUPS][G * V];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
#pragma unroll
    for (int v = 0; v < V; ++v) s_add[group][v * G + lane] = 0.0f;
    op_next_may_start();
    op_wait_for_previous();
    const float n = (float)max(*n_rows, 1);
    const float db = dlosses ? dlosses[0] : 0.0f, dz = dlosses ? dlosses[1] : 0.0f;
    const float hk = db * (float)experts / (n * (float)k) / n, zk = 2.0f * dz / n;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = route_expert<G, VEC>(v, lane);
        h[v] = e < experts ? hk * (float)counts[e] : 0.0f;
    }
    __syncwarp();
    const int64_t first = (int64_t)blockIdx.x * GROUPS + (threadIdx.x / 32) * (32 / G);
    for (int64_t base = first; base < rows; base += (int64_t)gridDim.x * GROUPS) {
        const int64_t row = base + group % (32 / G);
        const bool exists = row < rows;
        const bool in = exists && (!mask || mask[row]);
        OpRaw<T, VEC> raw[V / VEC];
        route_load<T, G, V, VEC>(logits + row * stride, in, experts, lane, raw);
        int at[SLOTS];
        float ga[SLOTS], dg[SLOTS], dot = 0.0f;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int j = s * G + lane;
            const bool mine = in && j < k;
            at[s] = mine ? index[row * k + j] : -1;
            const bool ok = at[s] >= 0 && at[s] < experts;
            ga[s] = ok ? gate[row * k + j] : 0.0f;
            dg[s] = ok && dgate ? dgate[row * k + j] : 0.0f;
            dot = fmaf(ga[s], dg[s], dot);
            if (!ok) at[s] = -1;
        }
        dot = op_group_sum<G>(dot);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (at[s] >= 0) s_add[group][at[s]] = ga[s] * (renormalise ? dg[s] - dot : dg[s]);
        float l[V], top = -INFINITY, total = 0.0f, ph = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] = raw[v / VEC].get(v % VEC);
            top = fmaxf(top, l[v]);  // leaves a NaN out, which the sums then bring in
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bool live = top > -INFINITY;
        const float top_l = live ? top : 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] = route_exp(l[v], top_l);
            total += l[v];
            ph = fmaf(l[v], h[v], ph);
        }
        total = op_group_sum<G>(total);
        live = live || total != total;  // NaN beside -inf alone
        total = live ? total : 1.0f;
        const float inv = 1.0f / total;
        ph = op_group_sum<G>(ph) * inv;
        const float shift = zk * (top_l + logf(total)) - ph - (renormalise ? 0.0f : dot);
        __syncwarp();
        T* out = dlogits + row * dstride;
#pragma unroll
        for (int c = 0; c < V / VEC; ++c) {
            const int e = c * G * VEC + lane * VEC;
            float add[VEC], t[VEC];
            constexpr int STEP = VEC < 4 ? VEC : 4;
#pragma unroll
            for (int i = 0; i < VEC; i += STEP) {
                float q[STEP];
                op_load<float, STEP>(&s_add[group][e + i], q);
#pragma unroll
                for (int r = 0; r < STEP; ++r) add[i + r] = q[r];
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[i] = live ? fmaf(l[c * VEC + i] * inv, h[c * VEC + i] + shift, add[i]) : 0.0f;
            if (exists && e < experts) op_store<T, VEC>(out + e, t);
        }
        __syncwarp();
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (at[s] >= 0) s_add[group][at[s]] = 0.0f;
        __syncwarp();
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
int64_t route_balance_bytes(int experts) { return (int64_t)((experts + 31) / 32) * 8; }
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
        constexpr bool S = (V) <= 8;                                                                                                            \
        auto kern = wide ? (S && k > 2 ? k_route_forward<T, G, V, VW, S> : k_route_forward<T, G, V, VW, false>)                                 \
                         : (S && k > 2 ? k_route_forward<T, G, V, 1, S> : k_route_forward<T, G, V, 1, false>);                                  \
        if (smem > 40000) op_note(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                          \
        op_launch_next(s, dim3((unsigned)blocks), dim3(ROUTE_THREADS), smem, kern, (const T*)logits, stride, mask, rows, experts, k, renormalise, index, gate, part);             \
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
        op_launch_next(s, dim3((unsigned)blocks), dim3(256), 0, kern, (const T*)logits, stride, mask, rows, experts, k, renormalise, index, gate, dgate, counts, n_rows, dlosses, \
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
    if (rows < 0 || rows > INT32_MAX || rows * k > INT32_MAX) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "rows must not be negative and rows * k below 2^31");
    if (rows > 0 && !logits) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_logits is NULL");
    if (rows > 1 && stride < experts) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the row stride must be at least experts");
    if ((uintptr_t)logits % size) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_logits must be aligned to its elements");
    return TB_OK;
}

}  // namespace

extern "C" int64_t tb_route_forward_workspace(int64_t rows, int experts) {
    if (rows < 0 || experts < 1 || experts > ROUTE_MAX_E) return TB_ERR_INVALID_ARGUMENT;
    return route_balance_bytes(experts) + ((int64_t)route_forward_blocks(rows, experts) * (2 * experts + 2) + 1) * 4;
}

extern "C" int tb_route_forward(const void* d_logits, int64_t stride, int type, int64_t rows, int experts, int k, int renormalise, const uint8_t* d_mask,
                                int32_t* d_index, float* d_gate, int32_t* d_counts, int32_t* d_rows, float* d_prob_mean, float* d_losses, void* d_work,
                                int64_t work_bytes, void* stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    const int rc = route_check(type, rows, experts, k, d_logits, stride, err, err_len);
    if (rc != TB_OK) return rc;
    if ((rows > 0 && (!d_index || !d_gate)) || !d_counts || !d_rows || !d_prob_mean || !d_losses)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "an output pointer is NULL");
    if (((uintptr_t)d_index | (uintptr_t)d_gate | (uintptr_t)d_counts | (uintptr_t)d_rows | (uintptr_t)d_prob_mean | (uintptr_t)d_losses) & 3)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "outputs must be aligned to their elements");
    const int64_t need = tb_route_forward_workspace(rows, experts);
    if (!d_work || work_bytes < need || ((uintptr_t)d_work & 7))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "the workspace must be aligned and hold %lld bytes (got %lld)", (long long)need, (long long)work_bytes);
    const int size = op_type_size(type);
    const OpRows xr = {d_logits, stride * size, rows, (int64_t)experts * size}, mask = op_vector(d_mask, rows, 1), ix = op_vector(d_index, rows * k), ga = op_vector(d_gate, rows * k),
                 co = op_vector(d_counts, experts), nr = op_vector(d_rows, 1), pm = op_vector(d_prob_mean, experts), lo = op_vector(d_losses, 2);
    if (op_meets(xr, {ix, ga, co, nr, pm, lo}) || op_meets(mask, {ix, ga, co, nr, pm, lo}) || op_meets(ix, {ga, co, nr, pm, lo}) || op_meets(ga, {co, nr, pm, lo}) ||
        op_meets(co, {nr, pm, lo}) || op_meets(nr, {pm, lo}) || op_meets(pm, {lo}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "a result overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int blocks = route_forward_blocks(rows, experts);
    RouteParts part;
    part.balance = static_cast<double*>(d_work);
    part.p = reinterpret_cast<float*>(static_cast<uint8_t*>(d_work) + route_balance_bytes(experts));
    part.c = reinterpret_cast<int*>(part.p + (size_t)blocks * experts);
    part.z = reinterpret_cast<float*>(part.c + (size_t)blocks * (experts + 1));
    part.ticket = reinterpret_cast<int*>(part.z + blocks);
    const bool wide = route_wide(d_logits, stride, experts, size);
#define ARGS s, d_logits, stride, d_mask, rows, experts, k, renormalise, d_index, d_gate, part, wide
    if (type == TB_TYPE_F32) route_forward_go<float>(ARGS);
    else if (type == TB_TYPE_F16) route_forward_go<__half>(ARGS);
    else route_forward_go<__nv_bfloat16>(ARGS);
#undef ARGS
    op_launch_next(s, dim3((unsigned)((experts + 31) / 32)), dim3(1024), 0, k_route_final, part, blocks, experts, k, d_counts, d_rows, d_prob_mean, d_losses);
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
    if ((uintptr_t)d_dlogits % op_type_size(type) ||
        ((uintptr_t)d_index | (uintptr_t)d_gate | (uintptr_t)d_dgate | (uintptr_t)d_counts | (uintptr_t)d_rows | (uintptr_t)d_dlosses) & 3)
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "tensors must be aligned to their elements");
    if (!op_apart(d_logits, 0, stride, d_dlogits, 0, dstride, 1, rows, experts, op_type_size(type))) return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dlogits overlaps d_logits in part");
    if (op_meets({d_dlogits, dstride * op_type_size(type), rows, (int64_t)experts * op_type_size(type)},
                 {op_vector(d_mask, rows, 1), op_vector(d_index, rows * k), op_vector(d_gate, rows * k), op_vector(d_dgate, rows * k), op_vector(d_counts, experts), op_vector(d_rows, 1),
                  op_vector(d_dlosses, 2)}))
        return op_report(err, err_len, TB_ERR_INVALID_ARGUMENT, "d_dlogits overlaps another tensor");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = route_wide(d_logits, stride, experts, op_type_size(type)) && route_wide(d_dlogits, dstride, experts, op_type_size(type));
#define ARGS s, d_logits, stride, d_mask, rows, experts, k, renormalise, d_index, d_gate, d_dgate, d_counts, d_rows, d_dlosses, d_dlogits, dstride, wide
    if (type == TB_TYPE_F32) route_backward_go<float>(ARGS);
    else if (type == TB_TYPE_F16) route_backward_go<__half>(ARGS);
    else route_backward_go<__nv_bfloat16>(ARGS);
#undef ARGS
    return op_launched(err, err_len);
}
