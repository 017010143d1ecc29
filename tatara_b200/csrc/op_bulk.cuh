// Rings of asynchronous copies from global to shared memory, one per warp (embed_kernels.cu): whole rows are on their way without registers.
#pragma once
#include "op_common.cuh"

namespace {

enum { BULK_COPY, BULK_END };
#ifndef BULK_WAIT_LIMIT  // tries before a wait gives up; the one at the end outlasts the others
#define BULK_WAIT_LIMIT(role) ((role) == BULK_END ? 1 << 22 : 1 << 20)
#endif

__device__ __forceinline__ unsigned bulk_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }

// K slots of SLOT bytes.  A copy is at most SLOT bytes, a multiple of 16, between 16-byte boundaries.  put and take are called by whole warps; a slot is taken again
// K copies later, after a __syncwarp() behind the last access to what it held.
template <int K, int SLOT>
struct BulkRing {
    unsigned slots, bars;
    unsigned put_count = 0, taken = 0;
    bool ok = true;  // the same in all lanes: no wait has run out
    // bars: [K], of this warp
    __device__ __forceinline__ BulkRing(const void* memory, uint64_t* barriers) : slots(bulk_smem(memory)), bars(bulk_smem(barriers)) {
        if ((threadIdx.x & 31) == 0) {
            for (int k = 0; k < K; ++k) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * k) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
    }
    __device__ __forceinline__ void put(const void* from, unsigned bytes) {
        if (!ok) return;
        if ((threadIdx.x & 31) == 0) {
            const unsigned k = put_count % K, bar = bars + 8 * k;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(slots + k * SLOT), "l"(from), "r"(bytes), "r"(bar) : "memory");
        }
        ++put_count;
    }
    __device__ __forceinline__ bool arrived(int limit) {
        const unsigned bar = bars + 8 * (taken % K), parity = taken / K & 1;
        for (int i = 0; i < limit; ++i) {
            unsigned there;
            asm volatile(
                "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(there)
                : "r"(bar), "r"(parity)
                : "memory");
            if (there) return true;
        }
        return false;
    }
    // the slot of the next copy, once it is there
    __device__ __forceinline__ unsigned take() {
        const unsigned k = taken % K;
        if (ok) ok = __all_sync(0xffffffffu, arrived(BULK_WAIT_LIMIT(BULK_COPY)));
        if (ok) ++taken;
        return k;
    }
    // Before the slots hold anything else, and before the block ends: nothing is on its way any more.  There is something only after a wait that has run out.
    __device__ __forceinline__ void end() {
        for (; taken < put_count; ++taken)
            if (!arrived(BULK_WAIT_LIMIT(BULK_END))) put_count = taken;  // not waited for again
    }
};

}  // namespace
