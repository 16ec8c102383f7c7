// prompt_attention.cu — causal attention over packed prompts.
#include "paged.cuh"
#include "row_attention.cuh"

namespace pf {

namespace {

struct PromptParams {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int* offsets;
    int n_seqs, n_tokens, n_heads, n_kv_heads;
    float scale;
    uint32_t* err;
};

// First and last row of sequence b; false where its offsets are not usable.
__device__ __forceinline__ bool seq_rows(const PromptParams& p, int b, int& first, int& end) {
    first = p.offsets[b];
    end = p.offsets[b + 1];
    if (first >= 0 && end >= first && end <= p.n_tokens) return true;
    latch(p.err, ERR_BOUNDS);
    return false;
}

// One warp a (row, head).
template <typename T, int HD>
__global__ void __launch_bounds__(256) prompt_rows_kernel(const PromptParams p) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, h = blockIdx.y, g = h / (p.n_heads / p.n_kv_heads);
    const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= p.n_tokens) return;
    int first = -1;
    for (int b = 0; b < p.n_seqs; b++) {
        int a, e;
        if (seq_rows(p, b, a, e) && a <= i && i < e) first = a;
    }
    if (first < 0) return;
    float q[N];
#pragma unroll
    for (int d = 0; d < N; d++) q[d] = (float)static_cast<const T*>(p.q)[i * p.q_stride + h * HD + lane + 32 * d] * p.scale;
    RowSoftmax<HD> s;
    for (int64_t j = first; j <= i; j++) {
        float k[N], v[N];
#pragma unroll
        for (int d = 0; d < N; d++) {
            k[d] = (float)static_cast<const T*>(p.k)[j * p.k_stride + g * HD + lane + 32 * d];
            v[d] = (float)static_cast<const T*>(p.v)[j * p.v_stride + g * HD + lane + 32 * d];
        }
        s.add(warp_dot(q, k), v);
    }
#pragma unroll
    for (int d = 0; d < N; d++)
        static_cast<T*>(p.out)[i * p.out_stride + h * HD + lane + 32 * d] = (T)(s.o[d] / s.l);
}

template <typename T>
pf_status launch_prompt(const PromptParams& p, int hd, cudaStream_t st) {
    const dim3 grid(ceil_div(p.n_tokens, 8), p.n_heads);
    if (hd == 64) prompt_rows_kernel<T, 64><<<grid, 256, 0, st>>>(p);
    else prompt_rows_kernel<T, 128><<<grid, 256, 0, st>>>(p);
    return launch_check("prompt_attention");
}

}  // namespace

}  // namespace pf

using namespace pf;

extern "C" pf_status pf_prompt_attention(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                         const void* v, int64_t v_stride, void* out, int64_t out_stride, int32_t dtype,
                                         const int32_t* offsets, int32_t n_seqs, int32_t n_tokens, int32_t n_heads,
                                         int32_t n_kv_heads, int32_t head_dim, float scale, void* stream) {
    PF_CHECK(dtype == PF_BF16 || dtype == PF_F16, "pf_prompt_attention: dtype %d is neither PF_BF16 nor PF_F16", dtype);
    PF_CHECK(head_dim == 64 || head_dim == 128, "pf_prompt_attention: head_dim %d is neither 64 nor 128", head_dim);
    PF_CHECK(n_seqs >= 0 && n_tokens >= 0, "pf_prompt_attention: %d sequences, %d tokens", n_seqs, n_tokens);
    PF_CHECK(n_kv_heads > 0 && n_heads > 0 && n_heads <= 65535 && n_heads % n_kv_heads == 0,
             "pf_prompt_attention: %d heads over %d kv heads", n_heads, n_kv_heads);
    PF_CHECK(scale > 0.0f && scale <= 3.402823466e38f, "pf_prompt_attention: scale must be positive and finite");
    const int64_t wq = (int64_t)n_heads * head_dim, wk = (int64_t)n_kv_heads * head_dim;
    PF_CHECK(q_stride >= wq && out_stride >= wq && k_stride >= wk && v_stride >= wk,
             "pf_prompt_attention: a stride is smaller than its row");
    PF_CHECK(((q_stride | k_stride | v_stride | out_stride) % 8) == 0 &&
                 (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16) == 0,
             "pf_prompt_attention: pointers and strides must be multiples of 16 bytes");
    PF_TRY(require_device());
    if (n_seqs == 0 || n_tokens == 0) return PF_OK;
    PF_CHECK(q && k && v && out && offsets, "pf_prompt_attention: null argument");
    PromptParams p{q, k, v, out, q_stride, k_stride, v_stride, out_stride, offsets, n_seqs, n_tokens, n_heads,
                   n_kv_heads, scale, device_error_flag()};
    return dtype == PF_BF16 ? launch_prompt<__nv_bfloat16>(p, head_dim, as_stream(stream))
                            : launch_prompt<__half>(p, head_dim, as_stream(stream));
}
