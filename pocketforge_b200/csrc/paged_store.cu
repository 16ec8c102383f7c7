// paged_store.cu — new keys and values into the pages of the paged cache.
//
// A row (token, kv head) is read once and written once: bound by HBM for a
// prompt, by two trips to memory for a step.  A CTA takes kTokens tokens; its
// warps first find each one's sequence (a 32-way search of the offsets: two
// rounds up to 1,024 sequences) and leave its place in shared memory, then
// every group of LPR lanes moves one row's key and value, 16 bytes a lane of
// each (fp32, head_dim 64: 16 lanes), the row's largest value found by
// shuffles.
//
// int8 rows are KVCache::quantize_row's (src/kv_cache.cpp:19-28): scale =
// amax / 127, code = round(x * (127 / amax)) with halves away from zero, each
// step rounded to fp32; scale 1 for a row of zeros.  A row that holds an
// infinity or NaN has no such scale: its scale is NaN, so that whatever reads
// it is NaN too, and its codes are zero.
#include "paged.cuh"

namespace pf {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 16;  // tokens a CTA takes

// Number of entries of off[0 .. n) that are <= x (they do not decrease), by a whole warp.
__device__ __forceinline__ int count_le(const int* off, int n, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;  // off[i] <= x for i < lo; > x for i >= hi
    while (hi - lo > 0) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step + step - 1;
        const bool le = at < hi && off[at] <= x;
        const int k = __popc(__ballot_sync(0xffffffffu, le));  // off does not decrease: the first k lanes
        lo += k * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    return (float)x;
}

template <typename ST, typename CT, int HD>
__global__ void __launch_bounds__(kThreads) store_kernel(const pf_paged_cache c, int layer, const ST* __restrict__ k,
                                                         int64_t k_stride, const ST* __restrict__ v, int64_t v_stride,
                                                         const int* __restrict__ offsets, int n_seqs, int n_tokens,
                                                         uint32_t* err) {
    constexpr int EPT = 16 / sizeof(ST);  // elements a lane
    constexpr int LPR = HD / EPT;         // lanes a row
    __shared__ int s_page[kTokens], s_slot[kTokens];
    const int t0 = blockIdx.x * kTokens, lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < kTokens; i += kThreads / 32) {
        const int t = t0 + i;
        int page = -1, slot = 0;
        if (t < n_tokens) {
            const int b = count_le(offsets, n_seqs + 1, t) - 1;
            if (b >= 0 && b < n_seqs) {
                const int n = seq_len(c, b, lane == 0 ? err : nullptr);
                const int64_t pos = (int64_t)n - ((int64_t)offsets[b + 1] - t);
                if (n >= 0 && pos >= 0 && pos < n) {
                    page = c.table[(int64_t)b * c.max_pages + pos / c.page_size];
                    slot = (int)(pos % c.page_size);
                }
                if ((unsigned)page >= (unsigned)c.n_pages) {
                    page = -1;
                    if (lane == 0) latch(err, ERR_BOUNDS);
                }
            }
        }
        if (lane == 0) s_page[i] = page, s_slot[i] = slot;
    }
    __syncthreads();
    const int G = c.n_kv_heads, part = threadIdx.x % LPR;
    for (int u = threadIdx.x / LPR; u < kTokens * G; u += kThreads / LPR) {  // uniform over the lanes of a row
        const int i = u / G, g = u % G, page = s_page[i];
        if (page < 0) continue;
        union {
            uint4 w;
            ST e[EPT];
        } x[2];
        x[0].w = *reinterpret_cast<const uint4*>(k + (t0 + i) * k_stride + g * HD + part * EPT);
        x[1].w = *reinterpret_cast<const uint4*>(v + (t0 + i) * v_stride + g * HD + part * EPT);
        const int64_t row = slot_row(c, page, layer, g, s_slot[i]);
        // the lanes of this row, all here
        const unsigned mask = (LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u)) << (lane & ~(LPR - 1));
#pragma unroll
        for (int w = 0; w < 2; w++) {
            CT* to = reinterpret_cast<CT*>(w ? c.v : c.k) + row * HD + part * EPT;
            union {
                CT e[EPT];
                uint32_t w32[EPT * sizeof(CT) / 4 > 0 ? EPT * sizeof(CT) / 4 : 1];
            } y;
            if constexpr (sizeof(CT) == 1) {
                float big = 0.0f;
                bool bad = false;
#pragma unroll
                for (int j = 0; j < EPT; j++) {
                    const float a = fabsf(to_float(x[w].e[j]));
                    bad |= !(a <= 3.402823466e38f);
                    big = fmaxf(big, a);
                }
                if (bad) big = __int_as_float(0x7f800000);
#pragma unroll
                for (int o = LPR / 2; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor_sync(mask, big, o));
                bad = big > 3.402823466e38f;
                const float scale = bad ? __int_as_float(0x7fffffff) : (big == 0.0f ? 1.0f : __fdiv_rn(big, 127.0f));
                const float mul = big == 0.0f ? 1.0f : __fdiv_rn(127.0f, big);
#pragma unroll
                for (int j = 0; j < EPT; j++)
                    y.e[j] = bad ? (CT)0 : (CT)(int)roundf(__fmul_rn(to_float(x[w].e[j]), mul));
                if (part == 0) (w ? c.v_scale : c.k_scale)[row] = scale;
            } else {
#pragma unroll
                for (int j = 0; j < EPT; j++) y.e[j] = (CT)to_float(x[w].e[j]);  // rounded to the nearest
            }
            constexpr int WORDS = EPT * sizeof(CT) / 4;
            if constexpr (WORDS == 4)
                *reinterpret_cast<uint4*>(to) = make_uint4(y.w32[0], y.w32[1], y.w32[2], y.w32[3]);
            else if constexpr (WORDS == 2)
                *reinterpret_cast<uint2*>(to) = make_uint2(y.w32[0], y.w32[1]);
            else
                *reinterpret_cast<uint32_t*>(to) = y.w32[0];
        }
    }
}

template <typename ST, typename CT>
pf_status launch_store(const pf_paged_cache& c, int layer, const void* k, int64_t ks, const void* v, int64_t vs,
                       const int* offsets, int n_seqs, int n_tokens, cudaStream_t st) {
    const int grid = ceil_div(n_tokens, kTokens);
    uint32_t* err = device_error_flag();
    const ST *kp = static_cast<const ST*>(k), *vp = static_cast<const ST*>(v);
    if (c.head_dim == 64)
        store_kernel<ST, CT, 64><<<grid, kThreads, 0, st>>>(c, layer, kp, ks, vp, vs, offsets, n_seqs, n_tokens, err);
    else
        store_kernel<ST, CT, 128><<<grid, kThreads, 0, st>>>(c, layer, kp, ks, vp, vs, offsets, n_seqs, n_tokens, err);
    return launch_check("paged_store");
}

}  // namespace

}  // namespace pf

using namespace pf;

extern "C" pf_status pf_paged_store(const pf_paged_cache* c, int32_t layer, const void* k, int64_t k_stride,
                                    const void* v, int64_t v_stride, int32_t dtype, const int32_t* offsets,
                                    int32_t n_seqs, int32_t n_tokens, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_store", false));
    PF_CHECK(layer >= 0 && layer < c->n_layers, "pf_paged_store: layer %d of %d", layer, c->n_layers);
    PF_CHECK(n_seqs >= 0 && n_seqs <= c->max_seqs && n_tokens >= 0, "pf_paged_store: %d sequences of %d, %d tokens",
             n_seqs, c->max_seqs, n_tokens);
    PF_CHECK(dtype == PF_F32 || (c->dtype == PF_I8 ? dtype == PF_BF16 || dtype == PF_F16 : dtype == c->dtype),
             "pf_paged_store: rows of dtype %d into a cache of dtype %d", dtype, c->dtype);
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim, es = type_bytes(dtype);
    PF_CHECK(k_stride >= width && v_stride >= width && k_stride * es % 16 == 0 && v_stride * es % 16 == 0 &&
                 (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0,
             "pf_paged_store: rows are narrower than the heads or not 16-byte aligned");
    PF_TRY(require_device());
    if (n_seqs == 0 || n_tokens == 0) return PF_OK;
    PF_CHECK(k && v && offsets, "pf_paged_store: null argument");
    cudaStream_t st = as_stream(stream);
    if (c->dtype == PF_I8) {
        if (dtype == PF_F32) return launch_store<float, int8_t>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
        if (dtype == PF_BF16) return launch_store<__nv_bfloat16, int8_t>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
        return launch_store<__half, int8_t>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
    }
    if (c->dtype == PF_BF16) {
        if (dtype == PF_F32) return launch_store<float, __nv_bfloat16>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
        return launch_store<__nv_bfloat16, __nv_bfloat16>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
    }
    if (dtype == PF_F32) return launch_store<float, __half>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
    return launch_store<__half, __half>(*c, layer, k, k_stride, v, v_stride, offsets, n_seqs, n_tokens, st);
}
