// paged.cuh — the paged cache (pf_paged_cache) as its kernels see it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace pf {

// Checks a cache's sizes, and its pointers as well (the page operations' `work`
// included with `need_work`); the message names the calling entry point.
pf_status check_paged_sizes(const pf_paged_cache* c, const char* where);
pf_status check_paged_cache(const pf_paged_cache* c, const char* where, bool need_work);

// What two launches of a page operation pass on, in the cache's `work`.
struct PageWork {
    int* n_list;   // pages in src / dst
    int* n_live;   // pages in use (compaction)
    int* src;      // [n_pages]
    int* dst;      // [n_pages]
    int* remap;    // [n_pages] of those at n_live and behind: new place of a page in use, -1 of a free one
    int* mark;     // [max_seqs] first list index that names the sequence
    int4* plan;    // [max_seqs] per list index: {pages asked for before it, its own, held}; of a fork, {fresh page, parent's page, length}
};
__host__ __device__ inline PageWork page_work(const pf_paged_cache& c) {
    int* w = reinterpret_cast<int*>(c.work);
    PageWork p;
    p.n_list = w;
    p.n_live = w + 1;
    p.plan = reinterpret_cast<int4*>(w + 4);
    p.src = w + 4 + 4 * (int64_t)c.max_seqs;
    p.dst = p.src + c.n_pages;
    p.remap = p.dst + c.n_pages;
    p.mark = p.remap + c.n_pages;
    return p;
}
inline size_t page_work_bytes(const pf_paged_cache& c) {
    return (4 + 3 * (size_t)c.n_pages + 5 * (size_t)c.max_seqs) * sizeof(int);
}

__host__ __device__ inline int type_bytes(int dtype) { return dtype == PF_F32 ? 4 : (dtype == PF_I8 ? 1 : 2); }
// Rows (page, layer, kv head, slot) are counted in 64 bits: a cache may hold more than 2^31 of them.
__device__ __forceinline__ int64_t slot_row(const pf_paged_cache& c, int page, int layer, int g, int slot) {
    return (((int64_t)page * c.n_layers + layer) * c.n_kv_heads + g) * c.page_size + slot;
}
__device__ __forceinline__ void latch(uint32_t* err, uint32_t bit) {
    if (err) atomicOr(err, bit);
}
// A sequence's length, -1 (and a latched bit) where it cannot be one.
__device__ __forceinline__ int seq_len(const pf_paged_cache& c, int b, uint32_t* err) {
    const int n = c.lens[b];
    if (n >= 0 && (int64_t)n <= (int64_t)c.max_pages * c.page_size) return n;
    latch(err, ERR_BOUNDS);
    return -1;
}

constexpr float kMaxScale = 2.3e38f;  // of scores: times log2 e it is still finite

constexpr int kDecide = 1024;  // threads of a CTA that decides for the others
// Exclusive prefix sum over the CTA's 1,024 threads, and the total.
__device__ __forceinline__ long long block_scan(long long v, long long* total, long long* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        long long w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    const long long before = warp ? s_warp[warp - 1] : 0;
    *total = s_warp[31];
    __syncthreads();  // s_warp is free for the next scan
    return before + x - v;
}

// A launch that may begin while the one before it in the stream still runs: the
// kernel waits for that one's end itself (after_previous) before it reads or
// writes anything, so only the way to its first instruction overlaps.
template <typename... P, typename... A>
pf_status launch_after(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                       A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PF_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return launch_check(what);
}
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace pf
