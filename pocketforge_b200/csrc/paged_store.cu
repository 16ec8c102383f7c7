// paged_store.cu — new keys and values into the pages of the paged cache.
//
// A row (token, kv head) is read once and written once: bound by HBM and the
// quantising for a prompt (23,000 tokens of 8 heads, fp32 to int8: 140 MB in 33
// us, 65% of the measured copy rate; bf16 to bf16 73%), by the chain of trips to
// memory (offsets, length, table, holders, row) for a step (320 tokens: 3.45 us).
// A CTA takes TOKENS tokens, as few as still fill the GPU; one of its warps finds
// their sequences (a 32-way search of the offsets for the first: two rounds up to
// 1,024 sequences; each of the others from there in doubling steps, which a
// million empty sequences between two tokens make 40 trips) and leaves their
// places in shared memory, while the others look at the offsets and the first
// rows are on their way.  Every group of head_dim / 8 lanes moves one row's key
// and value, 8 elements a lane of each (two contiguous runs of 4 if they are fp32), the
// row's largest value found by shuffles.  One row in flight a lane and more CTAs
// an SM: two or four rows in flight measured 5% and 35% slower on 64 prompts.  Quantising fp32 rows is as much work as moving them:
// the four quotients of a row (key and value, scale and multiplier) are made by
// four lanes, one each, and a code is rounded by adding 1.5 * 2^23 (to the
// nearest, ties to even) and putting the ties right.
//
// int8 rows are KVCache::quantize_row's (src/kv_cache.cpp:19-28): scale =
// amax / 127, code = round(x * (127 / amax)) with halves away from zero, each
// step rounded to fp32; scale 1 for a row of zeros.  A row that holds an
// infinity or NaN has no such scale: its scale is NaN, so that whatever reads
// it is NaN too, and its codes are zero.
#include <algorithm>

#include "paged.cuh"

namespace pf {

namespace {

constexpr int kThreads = 256;
constexpr int kElems = 8;  // elements a lane
constexpr int kLook = kThreads - 32;  // threads of a CTA that look at the offsets' order

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

// A lane's 8 elements: 8 at 8 * part, or (fp32) 4 at 4 * part of either half of the row, so that a group's loads are runs.
template <typename ST>
struct alignas(16) Piece {
    static constexpr int RUNS = sizeof(ST) / 2, RUN = kElems / RUNS;
    ST e[kElems];
};

// The largest magnitude of a row, inf if one is inf or NaN, in every lane of it.
template <typename ST, int LPR>
__device__ __forceinline__ float largest(const Piece<ST>& x, unsigned mask) {
    float big = 0.0f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kElems; j++) {
        const float a = fabsf((float)x.e[j]);
        bad |= !(a <= 3.402823466e38f);
        big = fmaxf(big, a);
    }
    if (bad) big = __int_as_float(0x7f800000);
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor_sync(mask, big, o));
    return big;
}

// round(x * mul) with halves away from zero, for |x * mul| <= 127 and a little, as four bytes.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float mul) {
    const float v[4] = {a, b, c, d};
    int r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = __fmul_rn(v[i], mul), m = fabsf(y), t = __fadd_rn(m, 12582912.0f);
        // m - round(m) is exact; 1/2 means a tie that went down to an even number
        const int n = __float_as_int(t) - __float_as_int(12582912.0f) + (__fsub_rn(m, __fsub_rn(t, 12582912.0f)) == 0.5f);
        r[i] = y < 0.0f ? -n : n;
    }
    uint32_t hi, all;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(r[3]), "r"(r[2]));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(all) : "r"(r[1]), "r"(r[0]), "r"(hi));
    return all;
}

// One row's key and value into the cache.
template <typename ST, typename CT, int HD>
__device__ __forceinline__ void put(const pf_paged_cache& c, int64_t row, const Piece<ST>& k, const Piece<ST>& v, int part,
                                    unsigned mask) {
    constexpr int LPR = HD / kElems;
    constexpr int RUNS = Piece<ST>::RUNS, RUN = Piece<ST>::RUN;
    CT* to_k = static_cast<CT*>(c.k) + row * HD + part * RUN;
    CT* to_v = static_cast<CT*>(c.v) + row * HD + part * RUN;
    if constexpr (sizeof(CT) == 1) {
        const float big_k = largest<ST, LPR>(k, mask), big_v = largest<ST, LPR>(v, mask);
        const float inf = __int_as_float(0x7f800000);
        // lane 0: k's scale, 1: v's, 2: k's multiplier, 3: v's.  127 / big is no number below 127 / FLT_MAX: such a row is
        // multiplied by 2^64 first.
        const float big = part & 1 ? big_v : big_k, up = big < 1e-36f ? 18446744073709551616.0f : 1.0f;
        float q = big == 0.0f ? 1.0f : (part & 2 ? __fdiv_rn(127.0f, big * up) : __fdiv_rn(big, 127.0f));
        if (!(part & 2) && big == inf) q = __int_as_float(0x7fffffff);
        if (part < 2) (part ? c.v_scale : c.k_scale)[row] = q;
        const int first = (threadIdx.x & 31) & ~(LPR - 1);
        const float mul_k = __shfl_sync(mask, q, first + 2), mul_v = __shfl_sync(mask, q, first + 3);
        auto codes = [&](const Piece<ST>& x, float big, float mul, CT* to) {
            uint2 w = make_uint2(0, 0);
            const float up = big < 1e-36f ? 18446744073709551616.0f : 1.0f;
            if (big < inf) {
                w.x = codes4((float)x.e[0] * up, (float)x.e[1] * up, (float)x.e[2] * up, (float)x.e[3] * up, mul);
                w.y = codes4((float)x.e[4] * up, (float)x.e[5] * up, (float)x.e[6] * up, (float)x.e[7] * up, mul);
            }
            if constexpr (RUNS == 1) *reinterpret_cast<uint2*>(to) = w;
            else *reinterpret_cast<uint32_t*>(to) = w.x, *reinterpret_cast<uint32_t*>(to + HD / 2) = w.y;
        };
        codes(k, big_k, mul_k, to_k);
        codes(v, big_v, mul_v, to_v);
    } else {
        Piece<CT> a, b;
#pragma unroll
        for (int j = 0; j < kElems; j++) a.e[j] = (CT)(float)k.e[j], b.e[j] = (CT)(float)v.e[j];  // to the nearest
        if constexpr (RUNS == 1) {
            *reinterpret_cast<uint4*>(to_k) = *reinterpret_cast<const uint4*>(&a);
            *reinterpret_cast<uint4*>(to_v) = *reinterpret_cast<const uint4*>(&b);
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                *reinterpret_cast<uint2*>(to_k + j * HD / 2) = reinterpret_cast<const uint2*>(&a)[j];
                *reinterpret_cast<uint2*>(to_v + j * HD / 2) = reinterpret_cast<const uint2*>(&b)[j];
            }
        }
    }
}

template <typename ST, typename CT, int HD, int TOKENS>
__global__ void __launch_bounds__(kThreads) store_kernel(const pf_paged_cache c, int layer, const ST* __restrict__ k,
                                                         int64_t k_stride, const ST* __restrict__ v, int64_t v_stride,
                                                         const int* __restrict__ offsets, int n_seqs, int n_tokens,
                                                         uint32_t* err) {
    constexpr int LPR = HD / kElems, GROUPS = kThreads / LPR;  // lanes a row, rows the CTA has in hand at once
    __shared__ int s_page[TOKENS], s_slot[TOKENS];
    after_previous();
    const int t0 = blockIdx.x * TOKENS, lane = threadIdx.x & 31, G = c.n_kv_heads, part = threadIdx.x % LPR;
    const int tokens = min(TOKENS, n_tokens - t0), rows = tokens * G;
    // the lanes of a row, which are all here or all not
    const unsigned mask = (LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u)) << (lane & ~(LPR - 1));
    int u = threadIdx.x / LPR, i = u / G, g = u - i * G;  // row u: token i of the CTA, kv head g
    Piece<ST> x, y;
    auto load = [&]() {
        using P = Piece<ST>;
        const ST* from_k = k + (t0 + i) * k_stride + g * HD + part * P::RUN;
        const ST* from_v = v + (t0 + i) * v_stride + g * HD + part * P::RUN;
#pragma unroll
        for (int j = 0; j < P::RUNS; j++) {
            reinterpret_cast<uint4*>(&x)[j] = *reinterpret_cast<const uint4*>(from_k + j * HD / 2);
            reinterpret_cast<uint4*>(&y)[j] = *reinterpret_cast<const uint4*>(from_v + j * HD / 2);
        }
    };
    if (u < rows) load();
    if (threadIdx.x < 32) {  // one search for the first token; the others' sequences are close behind, or far behind empty ones
        int b = tokens > 0 ? count_le(offsets, n_seqs + 1, t0) - 1 : 0;
        if (lane < tokens) {
            const int t = t0 + lane;
            auto begun = [&](int i) { return i <= n_seqs && offsets[i] <= t; };  // (b = -1: offsets[0] > t0)
            int step = 1;
            for (; begun(b + step); step *= 2) b += step;
            while (step /= 2)
                if (begun(b + step)) b += step;
            int page = -1, slot = 0;
            if (b >= 0 && b < n_seqs && offsets[b] <= t) {
                const int n = seq_len(c, b, err);
                const int64_t pos = (int64_t)n - ((int64_t)offsets[b + 1] - t);
                if (n >= 0 && pos >= 0 && pos < n) {
                    page = c.table[(int64_t)b * c.max_pages + pos / c.page_size];
                    slot = (int)(pos % c.page_size);
                }
                // (a page that others hold too is theirs as it is: the sequence got no room, or its length was lowered into it)
                if ((unsigned)page >= (unsigned)c.n_pages || c.refs[page] > 1) {
                    page = -1;
                    latch(err, ERR_BOUNDS);
                }
            }
            s_page[lane] = page, s_slot[lane] = slot;
        }
    } else {  // meanwhile the other warps look at a share of the offsets' order
        for (int64_t j = (int64_t)blockIdx.x * kLook + threadIdx.x - 32; j < n_seqs; j += (int64_t)gridDim.x * kLook)
            if (offsets[j] > offsets[j + 1]) latch(err, ERR_BOUNDS);
    }
    __syncthreads();
    while (u < rows) {
        if (s_page[i] >= 0) put<ST, CT, HD>(c, slot_row(c, s_page[i], layer, g, s_slot[i]), x, y, part, mask);
        u += GROUPS;
        for (g += GROUPS; g >= G; g -= G) i++;
        if (u < rows) load();
    }
}

template <typename ST, typename CT, int HD>
pf_status launch_store(const pf_paged_cache& c, int layer, const void* k, int64_t ks, const void* v, int64_t vs,
                       const int* offsets, int n_seqs, int n_tokens, cudaStream_t st) {
    uint32_t* err = device_error_flag();
    const ST *kp = static_cast<const ST*>(k), *vp = static_cast<const ST*>(v);
    // CTAs behind the tokens', if there are very many sequences, only look at offsets: eight a thread
    const int look = ceil_div(n_seqs, 8 * kLook);
    // 16 tokens a CTA share one round of searches, from one CTA an SM on; below that the chain of a single round is what counts
    // (fp32 to int8, 8 kv heads, us with 2 and with 16: 640 tokens 3.6 and 6.3, 2,560 6.9 and 7.4, 3,840 9.5 and 8.2, 9,472
    // 21.6 and 15.6; 2 kv heads: 640 3.5 and 3.8, 2,560 6.2 and 4.0, 9,472 18.1 and 5.8)
    if (n_tokens >= 16 * 148)
        return launch_after("paged_store", store_kernel<ST, CT, HD, 16>, dim3(std::max(ceil_div(n_tokens, 16), look)), kThreads, 0, st, c,
                            layer, kp, ks, vp, vs, offsets, n_seqs, n_tokens, err);
    return launch_after("paged_store", store_kernel<ST, CT, HD, 2>, dim3(std::max(ceil_div(n_tokens, 2), look)), kThreads, 0, st, c, layer,
                        kp, ks, vp, vs, offsets, n_seqs, n_tokens, err);
}

template <typename ST, typename CT>
pf_status launch_store(const pf_paged_cache& c, int layer, const void* k, int64_t ks, const void* v, int64_t vs,
                       const int* offsets, int n_seqs, int n_tokens, cudaStream_t st) {
    return c.head_dim == 64 ? launch_store<ST, CT, 64>(c, layer, k, ks, v, vs, offsets, n_seqs, n_tokens, st)
                            : launch_store<ST, CT, 128>(c, layer, k, ks, v, vs, offsets, n_seqs, n_tokens, st);
}

}  // namespace

}  // namespace pf

using namespace pf;

extern "C" pf_status pf_paged_store(const pf_paged_cache* c, int32_t layer, const void* k, int64_t k_stride,
                                    const void* v, int64_t v_stride, int32_t dtype, const int32_t* offsets,
                                    int32_t n_seqs, int32_t n_tokens, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_store", false));
    PF_CHECK(layer >= 0 && layer < c->n_layers, "pf_paged_store: layer %d of %d", layer, c->n_layers);
    PF_CHECK(n_seqs >= 0 && n_seqs <= c->max_seqs && n_tokens >= 0 && n_tokens <= 1 << 30, "pf_paged_store: %d sequences of %d, %d tokens",
             n_seqs, c->max_seqs, n_tokens);
    PF_CHECK(dtype == PF_F32 || (c->dtype == PF_I8 ? dtype == PF_BF16 || dtype == PF_F16 : dtype == c->dtype),
             "pf_paged_store: rows of dtype %d into a cache of dtype %d", dtype, c->dtype);
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim, es = type_bytes(dtype);
    PF_CHECK(k_stride >= width && v_stride >= width && k_stride * es % 16 == 0 && v_stride * es % 16 == 0 &&
                 (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0,
             "pf_paged_store: rows are narrower than the heads or not 16-byte aligned");
    PF_CHECK((uintptr_t)offsets % 4 == 0, "pf_paged_store: offsets must be 4-byte aligned");
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
