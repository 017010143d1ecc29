// Stable counting sort of entries by a small key, for the operators: entries by expert (expert_kernels.cu), tokens by a digit at a time (embed_kernels.cu).
//
//   count of key e, begin_e = sum of the counts before it (each rounded up to a multiple of `align`), place of entry i = begin_key(i) + how many
//   entries before i have its key.  Entries whose key is outside [0, E) have no place.
//
// A block of eight warps owns a piece of the entries, a warp an eighth of it.  First launch: the blocks' counts.  Last launch: every block adds up the counts
// ahead of its own, its warps count their eighths again into shared memory, turn the counts into places and walk their eighths once more, 32 entries at a time
// (a match over the warp's keys ranks them).  Where blocks times keys are many, a launch between the two adds the counts up once for all blocks; where all
// entries fit a block, the last launch is the only one.  No atomics on global memory, places do not depend on timing.
#pragma once
#include "op_common.cuh"

namespace {

#define SORT_THREADS 256
#define SORT_WARPS 8
#define SORT_MAX_E 1024
#define SORT_ONE 4096         // entries of a single block's sort
#define SORT_SCAN 16384       // blocks * keys above which a launch of its own adds up the counts

struct SortPlan {
    int blocks, keys, align;
    int64_t piece;            // entries per block
    bool scan;
};
inline SortPlan sort_plan(int64_t entries, int keys, int align) {
    SortPlan p;
    p.keys = keys;
    p.align = align;
    if (entries <= SORT_ONE) p.blocks = 1, p.piece = (entries > 0 ? entries + SORT_THREADS - 1 : SORT_THREADS) / SORT_THREADS * SORT_THREADS, p.scan = false;
    else {
        // as many blocks as there are SMs, of 1024 entries or more; more keys make every block's tables dearer
        const int64_t least = keys <= 64 ? 1024 : keys <= 512 ? 4096 : 8192, most = 2 * (int64_t)sm_count();
        const int64_t want = (entries + least - 1) / least, b = want < most ? want : most;
        p.piece = ((entries + b - 1) / b + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
        p.blocks = (int)((entries + p.piece - 1) / p.piece);
        p.scan = (int64_t)p.blocks * keys > SORT_SCAN;
    }
    return p;
}
// 32-bit words of workspace: the blocks' counts and, with a scan, the keys' counts
inline int64_t sort_words(const SortPlan& p) { return p.blocks == 1 ? 0 : ((int64_t)p.blocks + (p.scan ? 1 : 0)) * p.keys; }

// Walks the entries [from, to) of a warp, 32 at a time: f(entry, key or -1, lanes with the same key)
template <typename Key, typename F>
__device__ __forceinline__ void sort_walk(const Key& key, int keys, int64_t from, int64_t to, int lane, F f) {
    for (int64_t i0 = from; i0 < to; i0 += 32) {
        const int64_t i = i0 + lane;
        int e = i < to ? key(i) : -1;
        if ((unsigned)e >= (unsigned)keys) e = -1;
        f(i, e, __match_any_sync(0xffffffffu, e));
    }
}

template <typename Key>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(Key key, int64_t entries, SortPlan p, int* __restrict__ part) {
    extern __shared__ int s_count[];
    op_next_may_start();
    for (int e = threadIdx.x; e < p.keys; e += SORT_THREADS) s_count[e] = 0;
    __syncthreads();
    op_wait_for_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t first = (int64_t)blockIdx.x * p.piece + warp * (p.piece / SORT_WARPS), last = min(first + p.piece / SORT_WARPS, entries);
    sort_walk(key, p.keys, first, last, lane, [&](int64_t, int e, unsigned peers) {
        if (e >= 0 && lane == __ffs(peers) - 1) atomicAdd(&s_count[e], __popc(peers));
    });
    __syncthreads();
    for (int e = threadIdx.x; e < p.keys; e += SORT_THREADS) part[(int64_t)blockIdx.x * p.keys + e] = s_count[e];
}

// the counts of the blocks before each block, in place, and the keys' counts behind them; a warp per 32 keys, its lanes a key each
__global__ void __launch_bounds__(32) k_sort_scan(SortPlan p, int* __restrict__ part) {
    op_next_may_start();
    op_wait_for_previous();
    const int e = blockIdx.x * 32 + threadIdx.x;
    if (e >= p.keys) return;
    int run = 0;
    for (int b0 = 0; b0 < p.blocks; b0 += 16) {
        int c[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = b0 + i < p.blocks ? part[(int64_t)(b0 + i) * p.keys + e] : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (b0 + i < p.blocks) part[(int64_t)(b0 + i) * p.keys + e] = run;
            run += c[i];
        }
    }
    part[(int64_t)p.blocks * p.keys + e] = run;
}

// Where the experts begin from their counts, both [keys] in shared memory (s_begin[keys] too: the end), by all threads of the block
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

// Key: entry -> key; Put: put(entry, place) for every entry (-1: no place), and put.rest(...) by every block with the begins in shared memory
template <typename Key, typename Put>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_place(Key key, int64_t entries, SortPlan p, const int* __restrict__ part, Put put) {
    extern __shared__ int s_mem[];
    int *s_total = s_mem, *s_begin = s_total + p.keys, *s_next = s_begin + p.keys + 1;  // s_next: [SORT_WARPS][keys]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, keys = p.keys;
    op_next_may_start();
    for (int i = threadIdx.x; i < SORT_WARPS * keys; i += SORT_THREADS) s_next[i] = 0;
    __syncthreads();
    op_wait_for_previous();
    const int64_t first = (int64_t)blockIdx.x * p.piece + warp * (p.piece / SORT_WARPS), last = min(first + p.piece / SORT_WARPS, entries);
    int* next = s_next + warp * keys;
    sort_walk(key, keys, first, last, lane, [&](int64_t, int e, unsigned peers) {
        if (e >= 0 && lane == __ffs(peers) - 1) next[e] += __popc(peers);  // a warp's leaders have keys of their own
        __syncwarp();
    });
    __syncthreads();
    // a key's places: its begin, the blocks before this one, the warps before this one
    int ahead[SORT_MAX_E / SORT_THREADS];
#pragma unroll
    for (int i = 0; i < SORT_MAX_E / SORT_THREADS; ++i) {
        const int e = threadIdx.x + i * SORT_THREADS;
        ahead[i] = 0;
        if (e >= keys) continue;
        int total = 0;
        if (p.blocks == 1) {
            for (int w = 0; w < SORT_WARPS; ++w) total += s_next[w * keys + e];
        } else if (p.scan) {
            ahead[i] = part[(int64_t)blockIdx.x * keys + e];
            total = part[(int64_t)p.blocks * keys + e];
        } else {
#pragma unroll 8
            for (int b = 0; b < p.blocks; ++b) {
                const int c = part[(int64_t)b * keys + e];
                total += c;
                if (b < (int)blockIdx.x) ahead[i] += c;
            }
        }
        s_total[e] = total;
    }
    __syncthreads();
    sort_begins(s_total, s_begin, p);
#pragma unroll
    for (int i = 0; i < SORT_MAX_E / SORT_THREADS; ++i) {
        const int e = threadIdx.x + i * SORT_THREADS;
        if (e >= keys) continue;
        int run = s_begin[e] + ahead[i];
        for (int w = 0; w < SORT_WARPS; ++w) {
            const int c = s_next[w * keys + e];
            s_next[w * keys + e] = run;
            run += c;
        }
    }
    __syncthreads();
    sort_walk(key, keys, first, last, lane, [&](int64_t i, int e, unsigned peers) {
        int place = -1;
        if (e >= 0) place = next[e] + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && lane == __ffs(peers) - 1) next[e] += __popc(peers);
        __syncwarp();
        if (i < last) put(i, place);
    });
    put.rest(s_total, s_begin, p);
}

template <typename Key, typename Put>
void sort_launch(cudaStream_t s, const SortPlan& p, const Key& key, int64_t entries, int* work, const Put& put) {
    if (p.blocks > 1) {
        op_launch_next(s, dim3((unsigned)p.blocks), dim3(SORT_THREADS), (size_t)p.keys * 4, k_sort_count<Key>, key, entries, p, work);
        if (p.scan) op_launch_next(s, dim3((unsigned)((p.keys + 31) / 32)), dim3(32), 0, k_sort_scan, p, work);
    }
    // at most 40 KB: 1024 keys of eight warps and two tables
    op_launch_next(s, dim3((unsigned)p.blocks), dim3(SORT_THREADS), (size_t)((SORT_WARPS + 2) * p.keys + 1) * 4, k_sort_place<Key, Put>, key, entries, p, (const int*)work, put);
}

}  // namespace
