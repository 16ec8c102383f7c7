// row_attention.cuh — one query row against a run of entries, by one warp:
// the online softmax written down plainly.  The reference point of the tiled
// kernels and their way out where a tile cannot be multiplied whole.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace pf {

// Running softmax of one row; lane l holds output dims l, l + 32, ...
template <int HD>
struct RowSoftmax {
    static constexpr int N = HD / 32;
    float m = -INFINITY, l = 0.0f, o[N];
    __device__ RowSoftmax() {
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = 0.0f;
    }
    // One entry: score x (the same in every lane), value v.
    __device__ void add(float x, const float (&v)[N]) {
        const float m2 = fmaxf(m, x);
        if (x == -INFINITY) return;  // no weight, whatever the others are
        const float old = m == m2 ? 1.0f : expf(m - m2), p = expf(x - m2);
        m = m2;
        l = l * old + p;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = o[i] * old + p * v[i];
    }
};

// q . k over the warp, the same in every lane.
template <int N>
__device__ __forceinline__ float warp_dot(const float (&q)[N], const float (&k)[N]) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) x += q[i] * k[i];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

}  // namespace pf
