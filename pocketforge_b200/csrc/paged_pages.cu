// paged_pages.cu — the pages of the paged cache: reserve, free, fork, copy,
// compact.
//
// Each operation that takes pages decides in one CTA of 1,024 threads which
// ones (prefix sums over the list's needs and over the reference counts, so
// that the answer never depends on the order in which threads arrive), and a
// second launch on all SMs moves the bytes.  The deciding CTA reads the
// reference counts with every thread's share in flight at once; it is bound by
// its chain of trips to memory and block scans (4.6 to 7 us for 256 to 1,024
// pages).  The copies are bound by HBM: every thread has four 16-byte loads in
// flight (256 of 1,024 pages of 22 layers moved: 783 MB in 120 us, the measured
// copy rate; 128 last pages of forks, 98 MB in 21 us).
#include <climits>

#include "paged.cuh"

namespace pf {

namespace {

constexpr int kPerThread = 64;  // pages a thread takes at once at most (one bit each)
constexpr int kCopy = 256;      // threads of a copying CTA
constexpr int kMaxPages = 1 << 28, kMaxSeqs = 1 << 20;
constexpr int kVecs = 4;        // 16-byte vectors a thread has in flight

// This thread's pages [first, first + count) of the chunk at `base`, as a mask
// of those in use.
struct Share {
    int first, count;
    unsigned long long live;
};
__device__ __forceinline__ int share_size(int n_pages) {
    const int per = (n_pages + kDecide - 1) / kDecide;
    return min(kPerThread, (per + 3) & ~3);
}
__device__ __forceinline__ Share share_of(const pf_paged_cache& c, int64_t base, int per) {
    Share s;
    const int64_t first = base + (int64_t)threadIdx.x * per;
    s.first = (int)min(first, (int64_t)c.n_pages);
    s.count = (int)min((int64_t)per, (int64_t)c.n_pages - s.first);
    s.live = 0;
#pragma unroll 8
    for (int i = 0; i < s.count; i++) s.live |= (unsigned long long)(c.refs[s.first + i] > 0) << i;
    return s;
}
__device__ __forceinline__ unsigned long long ones(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1; }

// Writes the lowest free pages, `want` at most, to list[] in order; returns how many there are.
__device__ __forceinline__ int list_free(const pf_paged_cache& c, long long want, int* list, long long* s_warp) {
    long long found = 0;
    const int per = share_size(c.n_pages);
    for (int64_t base = 0; base < c.n_pages && found < want; base += (int64_t)per * kDecide) {
        const Share s = share_of(c, base, per);
        unsigned long long free_ = ~s.live & ones(s.count);
        long long total;
        long long rank = found + block_scan(__popcll(free_), &total, s_warp);
        for (; free_ && rank < want; free_ &= free_ - 1, rank++) list[rank] = s.first + __ffsll((long long)free_) - 1;
        found += total;
    }
    __syncthreads();  // list[] is read by other threads
    return (int)min(found, want);
}

__device__ __forceinline__ bool in_range(int i, int n) { return (unsigned)i < (unsigned)n; }

// mark[s] = the first index of list[] that names sequence s, for every s in it.
__device__ __forceinline__ void mark_first(const pf_paged_cache& c, const int* list, int n, int* mark) {
    for (int i = threadIdx.x; i < n; i += kDecide)
        if (in_range(list[i], c.max_seqs)) mark[list[i]] = INT_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kDecide)
        if (in_range(list[i], c.max_seqs)) atomicMin(&mark[list[i]], i);
    __syncthreads();
}

// Pages that sequence s of length n holds, `most` at most: those its length asks for, and behind them what it has taken for
// tokens that its owner has given back since by a lower length.  Every operation that adds pages leaves -1 behind the last one.
__device__ __forceinline__ int held_pages(const pf_paged_cache& c, int s, int n, int most) {
    int held = (int)(((int64_t)n + c.page_size - 1) / c.page_size);
    if (n)
        while (held < most && in_range(c.table[(int64_t)s * c.max_pages + held], c.n_pages)) held++;
    return held;
}

// {pages that entry i of a reserve asks for, pages that its sequence holds}; -1: refused (bit latched by the caller's second
// look).
__device__ __forceinline__ int2 reserve_need(const pf_paged_cache& c, const PageWork& w, const int* seqs,
                                             const int* counts, int i, uint32_t* err) {
    const int s = seqs[i];
    if (!in_range(s, c.max_seqs) || w.mark[s] != i || counts[i] < 0) {
        latch(err, ERR_BOUNDS);
        return make_int2(-1, 0);
    }
    const int n = seq_len(c, s, err);
    if (n < 0) return make_int2(-1, 0);
    const int64_t pages = ((int64_t)n + counts[i] + c.page_size - 1) / c.page_size;
    if (pages > c.max_pages) {
        latch(err, ERR_CONTEXT);
        return make_int2(-1, 0);
    }
    const int held = held_pages(c, s, n, (int)pages);
    return make_int2((int)pages - held, held);
}

__global__ void __launch_bounds__(kDecide) reserve_kernel(const pf_paged_cache c, const int* seqs, const int* counts,
                                                          int n, uint32_t* err) {
    after_previous();
    __shared__ long long s_warp[32];
    const PageWork w = page_work(c);
    mark_first(c, seqs, n, w.mark);
    long long want = 0;
    for (int base = 0; base < n; base += kDecide) {
        const int i = base + threadIdx.x;
        const int2 need = i < n ? reserve_need(c, w, seqs, counts, i, err) : make_int2(0, 0);
        long long total;
        const long long before = want + block_scan(max(need.x, 0), &total, s_warp);
        if (i < n) w.plan[i] = make_int4(need.x < 0 ? -1 : (int)min(before, (long long)INT_MAX), need.x, need.y, 0);
        want += total;
    }
    const int found = want > 0 ? list_free(c, min(want, (long long)c.n_pages), w.src, s_warp) : 0;
    __syncthreads();
    // one warp an entry: its pages are w.src[before .. before + need)
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < n; i += kDecide / 32) {
        const int4 plan = w.plan[i];
        const int before = plan.x, need = plan.y, held = plan.z;
        if (before < 0) continue;
        const int s = seqs[i];
        if (need && (int64_t)before + need > found) {
            if (lane == 0) latch(err, ERR_CONTEXT);
            continue;
        }
        for (int j = lane; j < need; j += 32) {
            const int p = w.src[before + j];
            c.table[(int64_t)s * c.max_pages + held + j] = p;
            c.refs[p] = 1;
        }
        if (lane == 0) {
            if (need && held + need < c.max_pages) c.table[(int64_t)s * c.max_pages + held + need] = -1;
            c.lens[s] += counts[i];
        }
    }
}

// One CTA a sequence; whoever takes its length first frees it, so one named
// twice is freed once.
__global__ void free_kernel(const pf_paged_cache c, const int* seqs, uint32_t* err) {
    after_previous();
    __shared__ int s_len, s_end;
    const int s = seqs[blockIdx.x];
    if (!in_range(s, c.max_seqs)) {
        if (threadIdx.x == 0) latch(err, ERR_BOUNDS);
        return;
    }
    if (threadIdx.x == 0) s_len = atomicExch(&c.lens[s], 0), s_end = INT_MAX;
    __syncthreads();
    if (s_len < 0 || s_len > (int64_t)c.max_pages * c.page_size) {
        if (threadIdx.x == 0) c.lens[s] = s_len, latch(err, ERR_BOUNDS);  // left as it is
        return;
    }
    if (s_len == 0) return;
    const int pages = (int)(((int64_t)s_len + c.page_size - 1) / c.page_size);
    int* row = c.table + (int64_t)s * c.max_pages;
    auto give = [&](int j, int p) {
        row[j] = -1;
        if (in_range(p, c.n_pages)) atomicSub(&c.refs[p], 1);
        else latch(err, ERR_BOUNDS);
    };
    const int whole = pages / (int)blockDim.x * blockDim.x;
    for (int j = threadIdx.x; j < whole; j += blockDim.x) give(j, row[j]);
    for (int j0 = whole;; j0 += blockDim.x) {  // up to the first entry behind the length that is no page (held_pages)
        const int j = j0 + threadIdx.x, p = j < c.max_pages ? row[j] : -1;
        if (j >= pages && !in_range(p, c.n_pages)) atomicMin(&s_end, j);
        __syncthreads();
        const int end = s_end;
        if (j < end) give(j, p);
        if (end <= j0 + (int)blockDim.x) break;
        __syncthreads();  // s_end has been read
    }
}

constexpr int kForkNone = -1, kForkRefused = -2;  // no partly filled page; left as it is

__global__ void __launch_bounds__(kDecide) fork_decide_kernel(const pf_paged_cache c, const int* parents,
                                                              const int* children, int n, uint32_t* err) {
    after_previous();
    __shared__ long long s_warp[32];
    const PageWork w = page_work(c);
    mark_first(c, children, n, w.mark);
    for (int i = threadIdx.x; i < n; i += kDecide)  // a parent is no entry's child
        if (in_range(parents[i], c.max_seqs)) w.mark[parents[i]] = -1;
    __syncthreads();
    long long want = 0;
    for (int base = 0; base < n; base += kDecide) {
        const int i = base + threadIdx.x;
        int need = 0;
        int4 plan = make_int4(kForkRefused, -1, 0, 0);
        if (i < n) {
            const int p = parents[i], k = children[i];
            bool ok = in_range(p, c.max_seqs) && in_range(k, c.max_seqs) && w.mark[k] == i && c.lens[k] == 0;
            if (ok) plan.z = seq_len(c, p, err), ok = plan.z >= 0;
            if (ok && plan.z % c.page_size) {
                plan.y = c.table[(int64_t)p * c.max_pages + plan.z / c.page_size];
                ok = in_range(plan.y, c.n_pages);
                need = ok;
            }
            if (ok) plan.x = kForkNone;
            else latch(err, ERR_BOUNDS);
        }
        long long total;
        const long long before = want + block_scan(need, &total, s_warp);
        if (need) plan.x = (int)before;
        if (i < n) w.plan[i] = plan;
        want += total;
    }
    const int found = want > 0 ? list_free(c, min(want, (long long)c.n_pages), w.src, s_warp) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kDecide) {  // (each thread its own)
        const int rank = w.plan[i].x;
        if (rank < 0) continue;
        if (rank >= found) {
            latch(err, ERR_CONTEXT);
            w.plan[i].x = kForkRefused;
        } else {
            const int page = w.src[rank];
            w.plan[i].x = page;
            c.refs[page] = 1;
        }
    }
}

// CTA (y, i): table row and reference counts of child i (y == 0), and its last
// page's positions of eight (layer, kv head) pairs, one a warp.
__global__ void __launch_bounds__(kCopy) fork_copy_kernel(const pf_paged_cache c, const int* parents,
                                                          const int* children, uint32_t* err) {
    after_previous();
    const int i = blockIdx.y;
    const int4 plan = page_work(c).plan[i];
    const int fresh = plan.x, len = plan.z, full = len / c.page_size, rest = len % c.page_size;
    if (fresh == kForkRefused) return;
    if (blockIdx.x == 0) {
        const int p = parents[i], k = children[i];
        const int* from = c.table + (int64_t)p * c.max_pages;
        int* to = c.table + (int64_t)k * c.max_pages;
        for (int j = threadIdx.x; j < full; j += kCopy) {
            const int page = from[j];
            to[j] = page;
            if (in_range(page, c.n_pages)) atomicAdd(&c.refs[page], 1);
            else latch(err, ERR_BOUNDS);
        }
        if (threadIdx.x == 0) {
            if (rest) to[full] = fresh;
            if (full + (rest > 0) < c.max_pages) to[full + (rest > 0)] = -1;
            c.lens[k] = len;
        }
    }
    if (!rest) return;
    const int lane = threadIdx.x & 31, pair = blockIdx.x * (kCopy / 32) + (threadIdx.x >> 5);
    if (pair >= c.n_layers * c.n_kv_heads) return;
    const int64_t a = slot_row(c, plan.y, 0, pair, 0), b = slot_row(c, fresh, 0, pair, 0);
    const int row = c.head_dim * type_bytes(c.dtype), vecs = rest * row / 16;
    const uint4* ka = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(c.k) + a * row);
    const uint4* va = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(c.v) + a * row);
    uint4* kb = reinterpret_cast<uint4*>(reinterpret_cast<char*>(c.k) + b * row);
    uint4* vb = reinterpret_cast<uint4*>(reinterpret_cast<char*>(c.v) + b * row);
    float sk[4], sv[4];  // 128 slots at most
    if (c.dtype == PF_I8) {
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (lane + 32 * u < rest) sk[u] = c.k_scale[a + lane + 32 * u], sv[u] = c.v_scale[a + lane + 32 * u];
    }
    for (int j = lane; j < vecs; j += 32 * kVecs) {
        uint4 x[kVecs], y[kVecs];
#pragma unroll
        for (int u = 0; u < kVecs; u++)
            if (j + 32 * u < vecs) x[u] = ka[j + 32 * u], y[u] = va[j + 32 * u];
#pragma unroll
        for (int u = 0; u < kVecs; u++)
            if (j + 32 * u < vecs) kb[j + 32 * u] = x[u], vb[j + 32 * u] = y[u];
    }
    if (c.dtype == PF_I8) {
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (lane + 32 * u < rest) c.k_scale[b + lane + 32 * u] = sk[u], c.v_scale[b + lane + 32 * u] = sv[u];
    }
}

// Copies whole pages src[i] -> dst[i], in pieces of kCopy * kVecs vectors.
__device__ __forceinline__ void copy_pages(const pf_paged_cache& c, const int* src, const int* dst, int n,
                                           uint32_t* err) {
    const int64_t rows = (int64_t)c.n_layers * c.n_kv_heads * c.page_size;
    const int64_t kv_vecs = rows * c.head_dim * type_bytes(c.dtype) / 16, sc_vecs = c.dtype == PF_I8 ? rows / 4 : 0;
    constexpr int piece = kCopy * kVecs;
    const int64_t kv_pieces = (kv_vecs + piece - 1) / piece, sc_pieces = (sc_vecs + piece - 1) / piece;
    const int64_t per = 2 * (kv_pieces + sc_pieces);
    for (int64_t u = blockIdx.x; u < per * n; u += gridDim.x) {
        const int i = (int)(u / per), from = src[i], to = dst[i];
        if (!in_range(from, c.n_pages) || !in_range(to, c.n_pages)) {
            if (threadIdx.x == 0) latch(err, ERR_BOUNDS);
            continue;
        }
        int64_t at = u % per;
        uint4* base;
        int64_t vecs;
        if (at < 2 * kv_pieces) {
            base = reinterpret_cast<uint4*>(at < kv_pieces ? c.k : c.v);
            vecs = kv_vecs;
            at %= kv_pieces;
        } else {
            at -= 2 * kv_pieces;
            base = reinterpret_cast<uint4*>(at < sc_pieces ? c.k_scale : c.v_scale);
            vecs = sc_vecs;
            at %= sc_pieces;
        }
        const uint4* a = base + from * vecs;
        uint4* b = base + to * vecs;
        const int64_t j = at * piece + threadIdx.x;
        uint4 x[kVecs];
#pragma unroll
        for (int q = 0; q < kVecs; q++)
            if (j + q * kCopy < vecs) x[q] = a[j + q * kCopy];
#pragma unroll
        for (int q = 0; q < kVecs; q++)
            if (j + q * kCopy < vecs) b[j + q * kCopy] = x[q];
    }
}

__global__ void __launch_bounds__(kCopy) copy_kernel(const pf_paged_cache c, const int* src, const int* dst, int n,
                                                     uint32_t* err) {
    after_previous();
    copy_pages(c, src, dst, n, err);
}

// n_live, the pages in use behind it (src) and the free ones before it (dst),
// pairwise; reference counts move with them.
__global__ void __launch_bounds__(kDecide) compact_decide_kernel(const pf_paged_cache c) {
    after_previous();
    __shared__ long long s_warp[32];
    const PageWork w = page_work(c);
    const int per = share_size(c.n_pages);
    const int64_t chunk = (int64_t)per * kDecide;
    const Share first = share_of(c, 0, per);  // all of them, up to 65,536 pages
    long long live = 0;
    for (int64_t base = 0; base < c.n_pages; base += chunk) {
        const Share s = base ? share_of(c, base, per) : first;
        long long total;
        block_scan(__popcll(s.live), &total, s_warp);
        live += total;
    }
    const int n_live = (int)live;
    long long holes = 0, movers = 0;
    for (int64_t base = 0; base < c.n_pages; base += chunk) {
        const Share s = base ? share_of(c, base, per) : first;
        // pages before n_live count if free, those behind it if in use
        const int front = min(max(n_live - s.first, 0), s.count);
        unsigned long long hole = ~s.live & ones(front), mover = s.live & ~ones(front);
        for (unsigned long long dead = ~s.live & ~ones(front) & ones(s.count); dead; dead &= dead - 1)
            w.remap[s.first + __ffsll((long long)dead) - 1] = -1;  // a table that names it is wrong
        long long total;
        const long long before =
            block_scan(((long long)__popcll(hole) << 32) | __popcll(mover), &total, s_warp);
        long long h = holes + (before >> 32), m = movers + (before & 0xffffffffll);
        for (; hole; hole &= hole - 1) w.dst[h++] = s.first + __ffsll((long long)hole) - 1;
        for (; mover; mover &= mover - 1) w.src[m++] = s.first + __ffsll((long long)mover) - 1;
        holes += total >> 32;
        movers += total & 0xffffffffll;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (int)movers; i += kDecide) {
        const int a = w.src[i], b = w.dst[i];
        c.refs[b] = c.refs[a];
        c.refs[a] = 0;
        w.remap[a] = b;
    }
    if (threadIdx.x == 0) *w.n_list = (int)movers, *w.n_live = n_live;
}

__global__ void __launch_bounds__(kCopy) compact_move_kernel(const pf_paged_cache c, uint32_t* err) {
    after_previous();
    const PageWork w = page_work(c);
    const int n = *w.n_list, n_live = *w.n_live;
    if (n == 0) return;  // in order already
    // tables: one warp a sequence
    for (int s = (int)(blockIdx.x * (kCopy / 32) + (threadIdx.x >> 5)); s < c.max_seqs; s += gridDim.x * (kCopy / 32)) {
        const int len = seq_len(c, s, err);
        const int pages = (int)(((int64_t)max(len, 0) + c.page_size - 1) / c.page_size);
        int* row = c.table + (int64_t)s * c.max_pages;
        auto follow = [&](int j, int p) {
            const int to = !in_range(p, c.n_pages) ? -1 : p < n_live ? p : w.remap[p];
            if (to < 0) latch(err, ERR_BOUNDS);
            else if (to != p) row[j] = to;
        };
        const int whole = pages & ~31;
        int j = threadIdx.x & 31;
        for (; j < whole; j += 32) follow(j, row[j]);
        for (bool more = pages > 0; more; j += 32) {  // the last ones, and those held behind the length
            const int p = j < c.max_pages ? row[j] : -1;
            const unsigned ends = __ballot_sync(0xffffffffu, j >= pages && !in_range(p, c.n_pages));
            more = ends == 0;
            if (more || (threadIdx.x & 31) < __ffs((int)ends) - 1) follow(j, p);
        }
    }
    copy_pages(c, w.src, w.dst, n, err);
}

constexpr int kCopyCtas = 148 * 8;  // all SMs full of copying CTAs

}  // namespace

pf_status check_paged_sizes(const pf_paged_cache* c, const char* where) {
    PF_CHECK(c, "%s: null cache", where);
    PF_CHECK(c->dtype == PF_I8 || c->dtype == PF_BF16 || c->dtype == PF_F16, "%s: cache dtype %d", where, c->dtype);
    PF_CHECK(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d is neither 64 nor 128", where, c->head_dim);
    PF_CHECK(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
             "%s: page_size %d is not 16, 32, 64 or 128", where, c->page_size);
    PF_CHECK(c->n_layers > 0 && c->n_kv_heads > 0 && c->n_pages > 0 && c->max_seqs > 0 && c->max_pages > 0,
             "%s: a size is not positive", where);
    PF_CHECK((int64_t)c->n_layers * c->n_kv_heads <= 65536 && c->n_pages <= kMaxPages && c->max_seqs <= kMaxSeqs &&
                 (int64_t)c->max_pages * c->page_size <= 1 << 30,
             "%s: a size is too large", where);
    return PF_OK;
}

pf_status check_paged_cache(const pf_paged_cache* c, const char* where, bool need_work) {
    PF_TRY(check_paged_sizes(c, where));
    PF_CHECK(c->k && c->v && c->table && c->lens && c->refs, "%s: null pointer in the cache", where);
    PF_CHECK(c->dtype != PF_I8 || (c->k_scale && c->v_scale), "%s: an int8 cache needs scales", where);
    PF_CHECK(!need_work || c->work, "%s: null work in the cache", where);
    const uintptr_t all = (uintptr_t)c->k | (uintptr_t)c->v | (need_work ? (uintptr_t)c->work : 0) |
                          (c->dtype == PF_I8 ? (uintptr_t)c->k_scale | (uintptr_t)c->v_scale : 0);
    PF_CHECK(all % 16 == 0, "%s: k, v, scales and work must be 16-byte aligned", where);
    PF_CHECK(((uintptr_t)c->table | (uintptr_t)c->lens | (uintptr_t)c->refs) % 4 == 0,
             "%s: table, lens and refs must be 4-byte aligned", where);
    return PF_OK;
}

}  // namespace pf

using namespace pf;

extern "C" {

size_t pf_paged_work_bytes(const pf_paged_cache* c) {
    return check_paged_sizes(c, "pf_paged_work_bytes") == PF_OK ? page_work_bytes(*c) : 0;
}

pf_status pf_paged_reserve(const pf_paged_cache* c, const int32_t* seqs, const int32_t* counts, int32_t n,
                           void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_reserve", true));
    PF_CHECK(n >= 0 && n <= c->max_seqs, "pf_paged_reserve: %d sequences of %d", n, c->max_seqs);
    PF_CHECK(((uintptr_t)seqs | (uintptr_t)counts) % 4 == 0, "pf_paged_reserve: seqs and counts must be 4-byte aligned");
    PF_TRY(require_device());
    if (n == 0) return PF_OK;
    PF_CHECK(seqs && counts, "pf_paged_reserve: null argument");
    return launch_after("reserve", reserve_kernel, dim3(1), kDecide, 0, as_stream(stream), *c, seqs, counts, n, device_error_flag());
}

pf_status pf_paged_free(const pf_paged_cache* c, const int32_t* seqs, int32_t n, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_free", false));
    PF_CHECK(n >= 0 && n <= c->max_seqs, "pf_paged_free: %d sequences of %d", n, c->max_seqs);
    PF_CHECK((uintptr_t)seqs % 4 == 0, "pf_paged_free: seqs must be 4-byte aligned");
    PF_TRY(require_device());
    if (n == 0) return PF_OK;
    PF_CHECK(seqs, "pf_paged_free: null argument");
    return launch_after("free", free_kernel, dim3(n), 128, 0, as_stream(stream), *c, seqs, device_error_flag());
}

pf_status pf_paged_fork(const pf_paged_cache* c, const int32_t* parents, const int32_t* children, int32_t n,
                        void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_fork", true));
    PF_CHECK(n >= 0 && n <= c->max_seqs && n <= 65535, "pf_paged_fork: %d children of %d sequences", n, c->max_seqs);
    PF_CHECK(((uintptr_t)parents | (uintptr_t)children) % 4 == 0, "pf_paged_fork: parents and children must be 4-byte aligned");
    PF_TRY(require_device());
    if (n == 0) return PF_OK;
    PF_CHECK(parents && children, "pf_paged_fork: null argument");
    uint32_t* err = device_error_flag();
    PF_TRY(launch_after("fork_decide", fork_decide_kernel, dim3(1), kDecide, 0, as_stream(stream), *c, parents, children, n, err));
    const dim3 grid(ceil_div(c->n_layers * c->n_kv_heads, kCopy / 32), n);
    return launch_after("fork_copy", fork_copy_kernel, grid, kCopy, 0, as_stream(stream), *c, parents, children, err);
}

pf_status pf_paged_copy(const pf_paged_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_copy", false));
    PF_CHECK(n >= 0 && n <= c->n_pages, "pf_paged_copy: %d pages of %d", n, c->n_pages);
    PF_CHECK(((uintptr_t)src | (uintptr_t)dst) % 4 == 0, "pf_paged_copy: src and dst must be 4-byte aligned");
    PF_TRY(require_device());
    if (n == 0) return PF_OK;
    PF_CHECK(src && dst, "pf_paged_copy: null argument");
    return launch_after("copy", copy_kernel, dim3(kCopyCtas), kCopy, 0, as_stream(stream), *c, src, dst, n, device_error_flag());
}

pf_status pf_paged_compact(const pf_paged_cache* c, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_compact", true));
    PF_TRY(require_device());
    PF_TRY(launch_after("compact_decide", compact_decide_kernel, dim3(1), kDecide, 0, as_stream(stream), *c));
    return launch_after("compact_move", compact_move_kernel, dim3(kCopyCtas), kCopy, 0, as_stream(stream), *c, device_error_flag());
}

}  // extern "C"
