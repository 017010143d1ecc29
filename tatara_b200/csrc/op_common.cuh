// Shared by the operators on the caller's device tensors (norm_kernels.cu, route_kernels.cu, orth_kernels.cu): element types,
// 16-byte vectors, group reductions and how an entry point reports an error.
#pragma once
#include "../../include/tatara_b200.h"
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <initializer_list>

static __device__ __forceinline__ float op_float(float v) { return v; }
static __device__ __forceinline__ float op_float(__half v) { return __half2float(v); }
static __device__ __forceinline__ float op_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> static __device__ __forceinline__ T op_round(float v);
template <> __device__ __forceinline__ float op_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half op_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 op_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N adjacent elements as one access: 16 bytes, or a single element where rows do not start on 16-byte boundaries
template <typename T, int N>
struct alignas(N * sizeof(T)) OpVec {
    T v[N];
};
template <typename T, int N>
static __device__ __forceinline__ void op_load(const T* p, float (&to)[N]) {
    const OpVec<T, N> u = *reinterpret_cast<const OpVec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = op_float(u.v[i]);
}
template <typename T, int N>
static __device__ __forceinline__ void op_store(T* p, const float (&from)[N]) {
    OpVec<T, N> u;
#pragma unroll
    for (int i = 0; i < N; ++i) u.v[i] = op_round<T>(from[i]);
    *reinterpret_cast<OpVec<T, N>*>(p) = u;
}

// N adjacent elements as they lie in memory, two 16-bit ones to a register (as an array of __half they would take one each)
template <typename T, int N>
struct OpRaw {
    static_assert(N * sizeof(T) == 2 || N * sizeof(T) == 4 || N * sizeof(T) == 8 || N * sizeof(T) == 16, "one access");
    static constexpr int WORDS = N * sizeof(T) >= 4 ? N * sizeof(T) / 4 : 1;
    unsigned w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
        if (N * sizeof(T) == 16) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            w[0] = u.x, w[1 % WORDS] = u.y, w[2 % WORDS] = u.z, w[3 % WORDS] = u.w;
        } else if (N * sizeof(T) == 8) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[0] = u.x, w[1 % WORDS] = u.y;
        } else if (N * sizeof(T) == 2) {
            w[0] = *reinterpret_cast<const unsigned short*>(p);
        } else {
            w[0] = *reinterpret_cast<const unsigned*>(p);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float get(int i) const;
};
template <typename T> static __device__ __forceinline__ float op_word(unsigned w, int half);
template <> __device__ __forceinline__ float op_word<float>(unsigned w, int) { return __uint_as_float(w); }
template <> __device__ __forceinline__ float op_word<__half>(unsigned w, int half) { return __half2float(__ushort_as_half((unsigned short)(half ? w >> 16 : w))); }
template <> __device__ __forceinline__ float op_word<__nv_bfloat16>(unsigned w, int half) { return __uint_as_float(half ? w & 0xffff0000u : w << 16); }
template <typename T, int N>
__device__ __forceinline__ float OpRaw<T, N>::get(int i) const { return sizeof(T) == 4 ? op_word<T>(w[i % WORDS], 0) : op_word<T>(w[i / 2], i & 1); }

// sum over aligned groups of G lanes, the same bits in every lane (halves are added in a fixed order)
template <int G>
static __device__ __forceinline__ float op_group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The first error of a call's launches, taken from what they return: the thread's last error may be one that somebody else has left, and stays as it is.
inline thread_local cudaError_t op_first_error = cudaSuccess;
static inline void op_note(cudaError_t e) {
    if (e == cudaSuccess) return;
    cudaGetLastError();  // ours, reported by op_launched
    if (op_first_error == cudaSuccess) op_first_error = e;
}

// Launches overlap, those of one call and those of calls that follow one another on a stream (programmatic dependent launch): every kernel may start before
// the one ahead of it has finished, and waits for it to end before it touches global memory.  That one has waited for those ahead of itself in the same way.
static __device__ __forceinline__ void op_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
static __device__ __forceinline__ void op_next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
static inline void op_launch_next(cudaStream_t s, dim3 grid, dim3 block, size_t smem, void (*kernel)(P...), A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    op_note(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

static inline int op_type_size(int type) { return type == TB_TYPE_F32 ? 4 : type == TB_TYPE_F16 || type == TB_TYPE_BF16 ? 2 : 0; }

// Whether a result may be written while an input of the same shape is read: both are the same memory, element by element, or have no element in
// common.  (Rows are taken in any order and a row is read before it is written, so anything between gives results that depend on the order.)
static inline bool op_apart(const void* in, int64_t in_batch, int64_t in_stride, const void* out, int64_t out_batch, int64_t out_stride, int64_t batch, int64_t rows, int64_t n, int size) {
    if (rows == 1) in_stride = out_stride = batch > 1 ? 0 : n;
    if (batch == 1) in_batch = out_batch = 0;
    const auto bytes = [=](int64_t b, int64_t r) { return (uintptr_t)((batch - 1) * b + (rows - 1) * r + n) * size; };
    const uintptr_t a = (uintptr_t)in, b = (uintptr_t)out;
    if (a + bytes(in_batch, in_stride) <= b || b + bytes(out_batch, out_stride) <= a) return true;
    if (in_stride != out_stride || in_batch != out_batch) return false;
    if (a == b) return true;
    // the same pitch: other columns of the same rows
    const int64_t pitch = rows == 1 ? in_batch : in_stride, d = (int64_t)(b - a);
    if (pitch == 0 || in_batch % pitch || d % size) return false;
    const int64_t at = ((d / size) % pitch + pitch) % pitch;
    return at >= n && pitch - at >= n;
}

// Rows in memory; a vector is a single one, and one that is not given is NULL.
struct OpRows {
    const void* p;
    int64_t stride, rows, bytes;  // stride and the length of a row in bytes
};
static inline OpRows op_vector(const void* p, int64_t count, int size = 4) { return {p, 0, 1, count * size}; }
// Whether rows have a byte in common with one of the vectors: the first row that ends behind a vector's begin, where it begins before the vector's end.
static inline bool op_meets(const OpRows& a, std::initializer_list<OpRows> vectors) {
    for (const OpRows& v : vectors) {
        if (!a.p || !v.p || v.bytes < 1) continue;
        const uintptr_t at = (uintptr_t)a.p, begin = (uintptr_t)v.p, bytes = (uintptr_t)a.bytes;
        const uintptr_t first = begin < at + bytes ? 0 : a.rows > 1 ? (begin - at - bytes) / (uintptr_t)a.stride + 1 : 1;
        if (first < (uintptr_t)a.rows && at + first * (uintptr_t)a.stride < begin + (uintptr_t)v.bytes) return true;
    }
    return false;
}

#if defined(__GNUC__)
__attribute__((format(printf, 4, 5)))
#endif
static inline int op_report(char* err, size_t err_len, int code, const char* fmt, ...) {
    if (err && err_len) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, err_len, fmt, ap);
        va_end(ap);
    }
    return code;
}
static inline int op_launched(char* err, size_t err_len) {
    const cudaError_t e = op_first_error;
    op_first_error = cudaSuccess;
    if (e == cudaSuccess) return TB_OK;
    return op_report(err, err_len, e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver ? TB_ERR_NO_DEVICE : TB_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
}
