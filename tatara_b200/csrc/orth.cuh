// Newton-Schulz orthogonalisation and the Muon step: what its two paths (orth_kernels.cu, orth_tc.cu) share.
//
//   u = the matrix (orthogonalise), or the momentum m' = beta m + g or g + beta m' (Muon, Nesterov)
//   X = u / (|u| + eps), transposed to n <= m;  `steps` times: A = X X^T, Q = a I + b A + c A^2, X = Q X
//   out = X (orthogonalise), or w' = clamp(w * w_mul - step * X) (Muon)
#pragma once
#include "op_common.cuh"

struct OrthIo {
    const void* g;                // [batch][rows][cols]
    int64_t g_batch, g_stride;
    const float* m;               // Muon: momentum, contiguous like w; NULL for orthogonalise
    float* m_out;
    float beta;
    int nesterov;
    void* out;                    // orthogonalise: of g's type; Muon: the new weights, fp32
    int64_t out_batch, out_stride;
    const float* w;
    float w_mul, step, clip;
    int rows, cols, batch;
};
struct OrthPoly {
    int steps;
    float a, b, c, eps;
};

// the new weight: w the old one, x the orthogonalised update
static __device__ __forceinline__ float orth_update(const OrthIo& io, float w, float x) {
    w = fmaf(-io.step, x, w * io.w_mul);
    w = w < -io.clip ? -io.clip : w;  // comparisons keep a NaN
    return w > io.clip ? io.clip : w;
}
// x is the result's element at that offset, w that of the old weights (Muon)
template <typename T>
static __device__ __forceinline__ void orth_store(const OrthIo& io, int64_t at, float w, float x) {
    if (!io.m) {
        static_cast<T*>(io.out)[at] = op_round<T>(x);
        return;
    }
    static_cast<float*>(io.out)[at] = orth_update(io, w, x);
}

// orth_kernels.cu: n <= ORTH_SMALL_N
#define ORTH_SMALL_N 64
void launch_orth_small(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int type);
// orth_tc.cu: any size; limbs: fp16 numbers that hold an operand (1: 11 bits, 2: 22 bits)
int64_t orth_tc_workspace(int batch, int rows, int cols, int limbs);
void launch_orth_tc(cudaStream_t s, const OrthIo& io, const OrthPoly& p, int type, int limbs, void* work);
