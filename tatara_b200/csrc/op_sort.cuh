// Stable counting sort of entries by a small key, for the operators: entries by expert (expert_kernels.cu), tokens by a digit at a time (embed_kernels.cu).
//
//   count of key e, begin_e = sum of the counts before it (each rounded up to a multiple of `align`), place of entry i = begin_key(i) + how many
//   entries before i have its key.  Entries whose key is outside [0, E) have no place.
//
// A block of eight warps owns a piece of the entries, a warp an eighth of it, 32 entries a step.  First launch: the blocks' counts.  Last launch: the warps count
// their eighths again into shared memory, every block adds up the counts ahead of its own, turns the counts into places, and its warps give every entry its own (votes over
// the warp's keys rank 32 entries at once).  Where blocks times keys are many, a launch between the two adds the counts up once for all
// blocks; where all entries fit a block, the last launch is the only one.  Places do not depend on timing.
//
// What bounds it is latency: an eighth's entries are loaded together (one step at a time cost a microsecond each) and stay in registers up to SORT_STEPS steps.
#pragma once
#include "op_common.cuh"

#include <type_traits>

namespace {

#define SORT_THREADS 256
#define SORT_WARPS 8
#define SORT_MAX_E 1024
#define SORT_STEPS 8          // of a warp, whose entries are in registers together
// entries of a single block's sort: 1200 x 1 of 9 4.0 us (two blocks 4.7), 2000 x 1 of 1024 5.8 (7.0), 3000 x 1 of 256 10.3 (several blocks 5.4); where `align` leaves much to fill it is slower (276 x 6 of 215, align 16: 10.5, several
// blocks 8.2)
#define SORT_ONE 2048
// Blocks * keys above which a launch of its own adds up the counts; with it and without, entries x keys: 80000 x 128 (10112) 8.2 and 7.0 us, 131072 x 128 (16384) 9.1 and 8.1, 320000 x 128 (20096) 11.7 and 11.6,
// 40000 x 512 (20480) 8.3 and 8.9, 80000 x 256 (20224) 9.0 and 10.5, 131072 x 256 (32768) 9.5 and 17.5.
#define SORT_SCAN 16384

struct SortPlan {
    int blocks, keys, align;
    int bits;                 // of a key
    int steps;                // of every warp; a block's piece is SORT_THREADS * steps entries
    bool scan;
};
// fill: places that may be left over, for the same blocks to fill
inline SortPlan sort_plan(int64_t entries, int keys, int align, int64_t fill = 0) {
    SortPlan p;
    p.keys = keys;
    p.align = align;
    for (p.bits = 0; 1 << p.bits < keys; ++p.bits) {}
    // four steps up to a block per SM, then up to SORT_STEPS with more blocks, then longer pieces
    const int64_t rows = (entries + SORT_THREADS - 1) / SORT_THREADS, sms = sm_count();
    int64_t steps = rows <= 4 * sms ? 4 : rows <= 2 * SORT_STEPS * sms ? SORT_STEPS : (rows + 2 * sms - 1) / (2 * sms);
    const bool one = entries <= SORT_ONE && fill <= 16 * SORT_ONE;
    if (one) steps = rows < 1 ? 1 : rows;
    else if (fill > 16 * SORT_ONE && rows < sms) steps = 1;
    p.steps = (int)steps;
    p.blocks = one || rows < 1 ? 1 : (int)((rows + steps - 1) / steps);
    p.scan = p.blocks > 1 && (int64_t)p.blocks * keys > SORT_SCAN;
    return p;
}
// 32-bit words of workspace: the blocks' counts and, with a scan, the keys' counts
inline int64_t sort_words(const SortPlan& p) { return p.blocks == 1 ? 0 : ((int64_t)p.blocks + (p.scan ? 1 : 0)) * p.keys; }

// The entries of a warp, S steps at a time.
template <typename Source, int S>
struct SortWalk {
    const Source& source;
    int keys, steps, bits, lane;
    int64_t first, entries;
    int v[S], id[S], rank[S];
    __device__ __forceinline__ SortWalk(const Source& src, int64_t n, const SortPlan& p)
        : source(src), keys(p.keys), steps(p.steps), bits(p.bits), lane(threadIdx.x & 31),
          first(((int64_t)blockIdx.x * SORT_WARPS + (threadIdx.x >> 5)) * p.steps * 32), entries(n) {}
    __device__ __forceinline__ void load(int s0) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int64_t i = first + (int64_t)(s0 + s) * 32 + lane;
            v[s] = -1, id[s] = 0;
            if (s0 + s < steps && i < entries) v[s] = source(i), id[s] = source.id(i);
        }
    }
    __device__ __forceinline__ int key(int s) const {
        const int e = source.key(v[s]);
        return (unsigned)e < (unsigned)keys ? e : -1;
    }
    // count[key] += 1 for every entry, in order; rank: what the count was before it.  The lanes with the same key are found by a vote per bit, all steps side by side (the match
    // instruction takes three times as long where keys differ).
    __device__ __forceinline__ void add(int* count) {
        unsigned peers[S];
        int before[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const unsigned any = __ballot_sync(0xffffffffu, key(s) >= 0);
            peers[s] = key(s) >= 0 ? any : ~any;
        }
        for (int b = 0; b < bits; ++b)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool one = key(s) >> b & 1;
                const unsigned set = __ballot_sync(0xffffffffu, one);
                peers[s] &= one ? set : ~set;
            }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            before[s] = 0;
            if (lane == __ffs(peers[s]) - 1 && key(s) >= 0) before[s] = atomicAdd(&count[key(s)], __popc(peers[s]));
            __syncwarp();  // another lane may add for the same key in the next step, and has to find this one's sum
        }
#pragma unroll
        for (int s = 0; s < S; ++s) rank[s] = __shfl_sync(0xffffffffu, before[s], __ffs(peers[s]) - 1) + __popc(peers[s] & ((1u << lane) - 1u));
    }
};

// zero: further words to be set to zero, for whoever counts into them later
template <typename Source, int S>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(Source source, int64_t entries, SortPlan p, int* __restrict__ part, int* __restrict__ zero, int64_t zeros) {
    extern __shared__ int s_count[];
    op_next_may_start();
    for (int e = threadIdx.x; e < p.keys; e += SORT_THREADS) s_count[e] = 0;
    __syncthreads();
    op_wait_for_previous();
    SortWalk<Source, S> w(source, entries, p);
    for (int s0 = 0; s0 < p.steps; s0 += S) {
        w.load(s0);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = w.key(s);
            if (e >= 0) atomicAdd(&s_count[e], 1);
        }
    }
    for (int64_t i = (int64_t)blockIdx.x * SORT_THREADS + threadIdx.x; i < zeros; i += (int64_t)gridDim.x * SORT_THREADS) zero[i] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < p.keys; e += SORT_THREADS) part[(int64_t)blockIdx.x * p.keys + e] = s_count[e];
}

// The counts of the blocks before each block, in place, and the keys' counts behind them.  A block per 32 keys, a lane per key, the warps a share of the blocks each.
__global__ void __launch_bounds__(1024) k_sort_scan(SortPlan p, int* __restrict__ part) {
    constexpr int U = 8;
    __shared__ int s_sum[32][32];
    op_next_may_start();
    op_wait_for_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int share = (p.blocks + 31) / 32, from = min(warp * share, p.blocks), to = min(from + share, p.blocks);
    int* at = part + (int64_t)from * p.keys + e;
    int sum = 0;
    for (int b0 = 0; b0 < to - from; b0 += U) {
        int c[U];
#pragma unroll
        for (int i = 0; i < U; ++i) c[i] = b0 + i < to - from && e < p.keys ? at[(int64_t)(b0 + i) * p.keys] : 0;
#pragma unroll
        for (int i = 0; i < U; ++i) sum += c[i];
    }
    s_sum[warp][lane] = sum;
    __syncthreads();
    int run = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) run += w < warp ? s_sum[w][lane] : 0;
    if (e >= p.keys) return;
    for (int b0 = 0; b0 < to - from; b0 += U) {
        int c[U];
#pragma unroll
        for (int i = 0; i < U; ++i) c[i] = b0 + i < to - from ? at[(int64_t)(b0 + i) * p.keys] : 0;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (b0 + i < to - from) at[(int64_t)(b0 + i) * p.keys] = run;
            run += c[i];
        }
    }
    if (warp == 31) part[(int64_t)p.blocks * p.keys + e] = run;
}

// Where the keys begin from their counts, both [keys] in shared memory (s_begin[keys] too: the end), by all threads of the block
__device__ __forceinline__ void sort_begins(const int* s_total, int* s_begin, const SortPlan& p) {
    __shared__ int s_warp[SORT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int PER = SORT_MAX_E / SORT_THREADS;
    int v[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = threadIdx.x * PER + i;
        v[i] = e < p.keys ? (s_total[e] + p.align - 1) / p.align * p.align : 0;
        sum += v[i];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += t;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += s_warp[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = threadIdx.x * PER + i;
        if (e <= p.keys) s_begin[e] = run;
        run += v[i];
    }
    if (threadIdx.x == SORT_THREADS - 1 && p.keys == SORT_MAX_E) s_begin[SORT_MAX_E] = run;
    __syncthreads();
}

// Source: the value and the identity of an entry, and the key in a value; Put: put(identity, value, place) for every entry (-1: no place), and put.rest(counts, begins, plan) by every block
template <typename Source, typename Put, int S>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_place(Source source, int64_t entries, SortPlan p, const int* part, Put put) {
    extern __shared__ int s_mem[];
    // s_total, s_ahead: a key's entries, those in the blocks before this one; s_next: [SORT_WARPS][keys]
    int *s_total = s_mem, *s_ahead = s_total + p.keys, *s_begin = s_ahead + p.keys, *s_next = s_begin + p.keys + 1;
    const int keys = p.keys;
    op_next_may_start();
    for (int i = threadIdx.x; i < 2 * keys; i += SORT_THREADS) s_total[i] = 0;
    for (int i = threadIdx.x; i < SORT_WARPS * keys; i += SORT_THREADS) s_next[i] = 0;
    op_wait_for_previous();
    SortWalk<Source, S> w(source, entries, p);
    w.load(0);
    __syncthreads();
    int* next = s_next + (threadIdx.x >> 5) * keys;
    if (p.blocks > 1 && p.scan) {
        for (int e = threadIdx.x; e < keys; e += SORT_THREADS) {
            s_ahead[e] = part[(int64_t)blockIdx.x * keys + e];
            s_total[e] = part[(int64_t)p.blocks * keys + e];
        }
    } else if (p.blocks > 1) {
        // keys side by side, the threads that are left share the blocks; U blocks' counts are on their way together, those behind the last whole batch too (10000 entries of 512 keys, ten
        // blocks: 6.4 us; with those behind it a load at a time 10.2)
        int width = 32;
        while (width < keys && width < SORT_THREADS) width *= 2;
        constexpr int U = 16;
        for (int e = threadIdx.x % width; e < keys; e += width) {
            const int step = SORT_THREADS / width;
            int total = 0, ahead = 0;
            int b0 = threadIdx.x / width;
            const auto batch = [&](auto whole) {
                int c[U];
#pragma unroll
                for (int i = 0; i < U; ++i) c[i] = decltype(whole)::value || b0 + i * step < p.blocks ? part[(int64_t)(b0 + i * step) * keys + e] : 0;
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    total += c[i];
                    if (b0 + i * step < (int)blockIdx.x) ahead += c[i];
                }
            };
            for (; b0 + (U - 1) * step < p.blocks; b0 += U * step) batch(std::true_type());
            if (b0 < p.blocks) batch(std::false_type());
            atomicAdd(&s_total[e], total);
            atomicAdd(&s_ahead[e], ahead);
        }
    }
    w.add(next);
    for (int s0 = S; s0 < p.steps; s0 += S) {
        w.load(s0);
        w.add(next);
    }
    __syncthreads();
    if (p.blocks == 1) {
        for (int e = threadIdx.x; e < keys; e += SORT_THREADS) {
            int total = 0;
#pragma unroll
            for (int k = 0; k < SORT_WARPS; ++k) total += s_next[k * keys + e];
            s_total[e] = total;
        }
        __syncthreads();
    }
    sort_begins(s_total, s_begin, p);
    // a key's places: its begin, the blocks before this one, the warps before this one
    for (int e = threadIdx.x; e < keys; e += SORT_THREADS) {
        int run = s_begin[e] + s_ahead[e];
#pragma unroll
        for (int k = 0; k < SORT_WARPS; ++k) {
            const int c = s_next[k * keys + e];
            s_next[k * keys + e] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int s0 = 0; s0 < p.steps; s0 += S) {
        const bool again = p.steps > S;  // counted on from the places themselves; otherwise the ranks are still there
        if (again) {
            w.load(s0);
            w.add(next);
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int64_t i = w.first + (int64_t)(s0 + s) * 32 + w.lane;
            const int e = w.key(s);
            if (s0 + s < p.steps && i < entries) put(w.id[s], w.v[s], e < 0 ? -1 : again ? w.rank[s] : next[e] + w.rank[s]);
        }
    }
    put.rest(s_total, s_begin, p);
}

// The launches of a sort: the blocks' counts into `part` (unless a sort before has counted them), then their sums and the places.
template <typename Source>
void sort_count(cudaStream_t s, const SortPlan& p, const Source& source, int64_t entries, int* part, int* zero = nullptr, int64_t zeros = 0) {
    if (p.blocks > 1)
        op_launch_next(s, dim3((unsigned)p.blocks), dim3(SORT_THREADS), (size_t)p.keys * 4, p.steps <= 4 ? k_sort_count<Source, 4> : k_sort_count<Source, SORT_STEPS>, source, entries, p, part, zero, zeros);
}
template <typename Source, typename Put>
void sort_place(cudaStream_t s, const SortPlan& p, const Source& source, int64_t entries, int* part, const Put& put) {
    if (p.scan) op_launch_next(s, dim3((unsigned)((p.keys + 31) / 32)), dim3(1024), 0, k_sort_scan, p, part);
    // at most 44 KB: 1024 keys of eight warps and three tables
    op_launch_next(s, dim3((unsigned)p.blocks), dim3(SORT_THREADS), (size_t)((SORT_WARPS + 3) * p.keys + 1) * 4, p.steps <= 4 ? k_sort_place<Source, Put, 4> : k_sort_place<Source, Put, SORT_STEPS>, source, entries,
                   p, (const int*)part, put);
}

}  // namespace
