// paged_attention.cu — attention of the newest tokens over the paged cache,
// split over the cache's length and joined.
//
//   out = sum_j softmax_j(scale * q . k_j) v_j   over the positions a row sees
//
// Every key and value is read once for all the query rows of its kv head (the
// group's heads times the newest tokens).  A (sequence, kv head, row group) is a
// segment of chunks (the warps' blocks side by side: 64 to 128 entries), cut into
// equal pieces of at most P chunks, one CTA a piece: where there are nearly as
// many segments as CTAs fit the GPU none is cut unless it is far longer than the
// others, and a few long ones are spread over every SM in one round.  The pieces
// of a cut segment are joined by the CTA that ends last, in their order (the
// answer does not depend on who that is).  Measured otherwise: one run of exactly
// total / CTAs chunks each, wherever it began and ended, 70 against 57 us on 64
// sequences of 512 to 1,024 with 5 rows (nearly every CTA had two segments to
// begin, end and join); pieces of half a share, 166 against 125 us on 8 contexts
// of 3,000 to 65,536 (a second round of CTAs, mostly empty); no limit to a
// segment's pieces, 115 against 21 us for one kv head's 30,000 entries (joining
// 235 of them).
//
// What bounds it (B200, measured): HBM for 16-bit caches (8 contexts of up to
// 65,536 entries, head_dim 128: 713 MB in 124 us, 5.7 TB/s, 88% of the measured
// copy rate); instruction issue for int8 ones, whose codes take one and a half
// instructions each on the way to an operand (16 contexts of 8,000, one fp32 row:
// 139 MB in 40.6 us, 53%); the chain of trips to memory before the first block
// and the joining for one short context (777 entries: 8.5 us).  64 sequences with
// 5 fp32 rows, 35 us for 55 MB: 20 rows make 24 columns and two planes of each,
// about 1,100 instructions a warp and 32 entries, issued at 0.44 a clock by the 10
// of 12 warps that are there on average (ncu; the tensor pipe is active in 29% of
// the cycles), a quarter of a CTA's time before its
// first block.
//
// A CTA's three (64-byte rows) or four warps take blocks of 32 entries (256-byte
// rows: 16) in turn, each with its own ring of them in flight (cp.async, no
// barrier between warps) and its own running softmax, and are put together at the
// end.  Three warps let 64-byte rows have four CTAs an SM: 592, so that the 512
// segments of 64 sequences and 8 kv heads run at once (55 to 45 us).  The
// products are 16x8x16 tensor-core ones with the entries (S^T = K Q^T) and the
// dims (O^T = V^T P^T) as the 16 and the query rows as the 8, so a few rows
// waste little; which entry or dim stands where in an operand is free as long
// as both operands agree, and is chosen so that every thread reads 16 (int8
// head_dim 64 values: 8) bytes of a stored row at a time, in banks apart.  The
// transposition that V needs is a byte permutation of two entries' words.
//
// Accuracy.  int8 codes are exact in fp16, and fp32 queries are split into two
// fp16 planes (22 bits) after a power of two takes the row's largest value to
// 2^13..2^14.  Over an int8 cache weights are two fp16 planes as well; they take
// the entry's scale, and a power of two that keeps a block's largest below 2^15.
// Over a 16-bit cache both operands of a product have its type.  With one column
// tile, where HBM is waited for, weights are two planes of it (64 x 1 rows at
// head_dim 128 38.1 and 38.6 us, 8 long contexts 124.5 and 125.6): the first is
// cut, not rounded, so that the second is above 0 as well and an inf among the
// values stays one.  With more tiles they are rounded to one plane, an error like
// the output's own rounding; a second one took 64 x 5 rows from 31.6 to 36.4 us
// (head_dim 64) and from 49.7 to 56.1 (128).  fp16 ends at 2^-24, and a
// long row's many weights below that can be its answer where the largest ones
// meet small values.  So the largest weights are taken to the end of fp16's range
// (LIFT, or the scales' power of two), and the maximum that exponents refer to
// rises as soon as it is exceeded by 2^6: a weight is off by 2^-34 of the row's
// largest at most beside its rounding (2^-33 where its second plane is kept above
// 0), over an int8 cache by 2^-33 of the largest weight times the largest scale of
// its block or of one before.  Rising from 2^2 on keeps four bits more but took 64 sequences
// with 5 rows from 35.2 to 38.8 us (int8) and 51.1 to 58.7 (fp16, head_dim 128);
// 2^6: 35.5 and 51.2.  bf16 has fp32's range: 2^8.  A block's products start from
// zero and are added to O in fp32 with rounding, as the tensor cores cut sums off
// instead, which would add up over a long cache.
//
// A row sees nothing behind its own position: those entries' weights are 0 by
// selection, entries behind the sequence's end are zeros in shared memory, and
// a 16-bit cache's last block is multiplied once for each new token with the
// values it may not see set to 0 (0 x inf would be NaN).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged.cuh"

namespace pf {

namespace {

constexpr int kMaxHeads = 65535;
constexpr int kMaxCuts = 64;     // pieces of a segment: as many as one CTA joins in about a microsecond
// Sequences from which on a launch of one CTA plans the pieces for all: its 2 us are less than what every CTA would take to
// look through them (bf16: 1,000 sequences of 50 to 200 tokens 314 and 121 us, 250 of them 49 and 35, 128 36.0 and 36.9; one kv
// head's 128 of 500 to 1,500, where the pieces are tried out, 22.6 and 20.0, 64 of them 16.5 and 18.0).
constexpr int kPlanned = 160, kPlannedFew = 96;
constexpr int kWhole = 4;        // chunks that are not cut if no sequence has more: joining costs 2 us (4 x 300 entries: 5.5 and 7.2 us)
constexpr int kCounters = 1024;  // at the start of `work`: seg_begin / P is below the CTAs that fit

struct PagedParams {
    pf_paged_cache c;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int layer, n_seqs, rows, n_heads, dtype;
    int group, cols, row_groups, page_shift;  // heads a kv head; rows x group; tiles of them; log2 page_size
    float scale;
    int ctas;      // that fit the GPU
    int* count;    // [kCounters] pieces of a cut segment that have ended
    int4* plan;    // of many sequences: {pieces, most}, then each piece's {sequence, which of its pieces, chunks before it, length}
    float* part;   // [piece of a cut segment][columns a row group][head_dim + 4]
    uint32_t* err;
};

// CTAs that fit an SM, by the bytes of a stored row, its type and the column tiles.  (Three with rings of two blocks instead of
// two of three, where the registers allow it: 1,000 sequences of 50 to 200 tokens 114 to 86 us, 16 of 8,000 49.1 to 48.2.)
__host__ __device__ constexpr int ctas_per_sm(int row_bytes, bool i8, int tiles) {
    return row_bytes == 64 ? 4 : (row_bytes == 128 && !i8 && tiles == 1 ? 3 : 2);
}

template <typename CT, int HD, int NT>
struct Ring {
    static constexpr int RB = HD * (int)sizeof(CT);                 // bytes of a stored row
    static constexpr int WARPS = RB == 64 ? 3 : 4;
    static constexpr int BLOCK = RB == 256 ? 16 : 32;               // entries a warp takes at a time
    static constexpr int CHUNK = WARPS * BLOCK;                     // entries the CTA takes at a time
    static constexpr int SCALES = sizeof(CT) == 1 ? 2 * BLOCK * 4 : 0;
    static constexpr int BYTES = 2 * BLOCK * RB + SCALES;           // keys, values, scales of a block
    static constexpr int CTAS = ctas_per_sm(RB, sizeof(CT) == 1, NT);
    static constexpr int STAGES = RB == 64 && NT == 1 ? 4 : (CTAS == 3 ? 2 : 3);
    static constexpr int SMEM = WARPS * STAGES * BYTES;
};

// Where 16-byte piece c of row r lies: rows read together in other banks.
template <int RB>
__device__ __forceinline__ int key_at(int r, int c) {
    return RB == 64 ? r * RB + c * 16 : r * RB + (c ^ ((r & 1) << 2)) * 16;
}
template <int RB>
__device__ __forceinline__ int value_row(int r) {
    return RB == 64 ? (r & ~3) | ((r & 1) << 1) | ((r >> 1) & 1) : r;
}
template <int RB>
__device__ __forceinline__ int value_at(int r, int c) {
    const int at = value_row<RB>(r);
    return RB == 64 ? at * RB + (c ^ (((at >> 2) & 1) << 1)) * 16 : at * RB + (c ^ (((r >> 1) & 3) << 1)) * 16;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
template <bool BF>
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two bytes (already +128) of x in halves: 0x6400 + u is 1024 + u in fp16.
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t x, uint32_t sel) {
    const uint32_t h = __byte_perm(x, 0x64646464u, sel);
    const __half2 y = __hsub2(reinterpret_cast<const __half2&>(h), __half2half2(__ushort_as_half(0x6480)));  // 1152
    return reinterpret_cast<const uint32_t&>(y);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if constexpr (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// The same, cut off instead of rounded.
template <bool BF>
__device__ __forceinline__ uint32_t pack_cut(float lo, float hi) {
    if constexpr (BF) return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// The same to fp16 with an inf taken down to the largest value.
__device__ __forceinline__ uint32_t pack_finite(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF>
__device__ __forceinline__ float2 unpack(uint32_t x) {
    if constexpr (BF) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    else return __half22float2(reinterpret_cast<const __half2&>(x));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^k for k in [-126, 127], as a float.
__device__ __forceinline__ float power_of_two(int k) { return __int_as_float((k + 127) << 23); }
// floor(log2 x) of a finite x > 0 (-127 for subnormal ones).
__device__ __forceinline__ int exponent_of(float x) { return (__float_as_int(x) >> 23) - 127; }

// 16 values from element i on (16-byte aligned): fp32 (two planes) or a 16-bit type.
template <int PLANES>
__device__ __forceinline__ void load16(const void* q, int64_t i, int dtype, bool on, float* v) {
    if constexpr (PLANES == 2) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float4 x = on ? reinterpret_cast<const float4*>(static_cast<const float*>(q) + i)[k] : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * k] = x.x, v[4 * k + 1] = x.y, v[4 * k + 2] = x.z, v[4 * k + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint4 x = on ? reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + i)[k] : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 y = dtype == PF_BF16 ? unpack<true>(w[e]) : unpack<false>(w[e]);
                v[8 * k + 2 * e] = y.x, v[8 * k + 2 * e + 1] = y.y;
            }
        }
    }
}
// A sequence's length as it counts here, and its chunks (one even if it is empty: its rows are zeros).
__device__ __forceinline__ int length_of(const PagedParams& p, int b, uint32_t* err) { return max(seq_len(p.c, b, err), 0); }
template <int CHUNK>
__device__ __forceinline__ int chunks_of(int len) {
    return max((len + CHUNK - 1) / CHUNK, 1);
}

// Pieces of at most `most` chunks that n are cut into (inv = 1 / most; n is exact in fp32), kMaxCuts at most.
__device__ __forceinline__ int cuts_of(int n, int most, float inv) {
    int k = (int)((float)n * inv);
    k += (k + 1) * most <= n;
    k -= k * most > n;                 // n / most
    return min(k + (k * most < n), kMaxCuts);
}

// Chunks a piece.  With nearly as many segments as CTAs fit, only what is twice as long as the share is cut.  With fewer, the
// least with which all pieces are there at once (a second, nearly empty round of CTAs costs more than pieces that are a little
// longer), of 32 between the share and twice that: pieces_at(most, 1 / most) says how many there are, fewer of longer ones.
// (int8, one fp32 row, 592 places; us with the border at 1/2, 3/4 and 1 of them: 320 segments of 500 to 1,500 entries 21.5, 22.0 and
// 22.0, 384: 23.7, 22.9 and 22.9, 512: 26.8, 26.8 and 27.6, 576: 28.0, 28.0 and 31.7; 384 of 4,000 63.5, 65.3 and 65.0, 576: 68.5, 68.5
// and 72.8.)
__host__ __device__ constexpr int few_segments(int ctas) { return ctas / 4 * 3; }
template <typename F>
__device__ __forceinline__ int piece_limit(int total, int segments, int ctas, const F& pieces_at) {
    const int share = (total + ctas - 1) / ctas, step = (share + 31) / 32;
    if (segments >= few_segments(ctas)) return 2 * share;
    int i = 0;
#pragma unroll 1
    for (int by = 16; by; by >>= 1) {
        const int mine = share + (i + by - 1) * step;
        if (pieces_at(mine, 1.0f / (float)mine) > ctas) i += by;
    }
    return share + i * step;
}

// x / group for a column x of at most eight tokens.
__device__ __forceinline__ int token_of(int x, int group) {
    int t = 0;
#pragma unroll
    for (int k = 1; k < 8; k++) t += x >= k * group;
    return t;
}

// Dims d, d + 1 of column x of kv head g: head g * group + x % group of token x / group.
__device__ __forceinline__ void store_out(const PagedParams& p, int seq, int g, int x, int d, int hd, float2 v) {
    const int token = token_of(x, p.group), head = g * p.group + x - token * p.group;
    const int64_t at = ((int64_t)seq * p.rows + token) * p.out_stride + head * hd + d;
    if (p.dtype == PF_F32) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at) = v;
    else
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at) =
            p.dtype == PF_BF16 ? pack<true>(v.x, v.y) : pack<false>(v.x, v.y);
}

// Sum over the CTA's threads, in all of them.
__device__ __forceinline__ int block_sum(int v, int* s_warp) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) s_warp[warp] = v;
    __syncthreads();
    v = __reduce_add_sync(0xffffffffu, s_warp[lane]);
    __syncthreads();
    return v;
}

// The plan of many sequences, which every CTA of the attention would take longer to make than to look up.
__global__ void __launch_bounds__(kDecide) plan_kernel(const PagedParams p, int chunk) {
    after_previous();
    __shared__ int s_sum[32];
    __shared__ long long s_scan[32];
    const int segs = p.c.n_kv_heads * p.row_groups;
    auto chunks = [&](int b, uint32_t* err) { return max((length_of(p, b, err) + chunk - 1) / chunk, 1); };
    int total = 0;
    bool long_one = false;
    for (int b = threadIdx.x; b < p.n_seqs; b += kDecide) {
        const int n = chunks(b, p.err);
        total += n;
        long_one |= n > kWhole;
    }
    total = block_sum(total, s_sum) * segs;
    const int most = !__syncthreads_or(long_one) ? kWhole : piece_limit(total, p.n_seqs * segs, p.ctas, [&](int mine, float inv) {
        int pieces = 0;
        for (int b = threadIdx.x; b < p.n_seqs; b += kDecide) pieces += cuts_of(chunks(b, nullptr), mine, inv);
        return block_sum(pieces, s_sum) * segs;
    });
    const float inv = 1.0f / (float)most;
    long long before = 0;  // pieces and chunks, 32 bits each
    for (int b0 = 0; b0 < p.n_seqs; b0 += kDecide) {
        const int b = b0 + threadIdx.x, n = b < p.n_seqs ? chunks(b, nullptr) : 0;
        long long all;
        const int my_pieces = n ? cuts_of(n, most, inv) * segs : 0;
        const long long x = before + block_scan(((long long)my_pieces << 32) | (n * segs), &all, s_scan);
        const int len = n ? length_of(p, b, nullptr) : 0;
        for (int i = 0; i < my_pieces; i++) p.plan[1 + (x >> 32) + i] = make_int4(b, i, (int)x, len);
        before += all;
    }
    if (threadIdx.x == 0) p.plan[0] = make_int4((int)(before >> 32), most, 0, 0);
}

template <typename CT, int HD, int NT, int PLANES>
__global__ void __launch_bounds__(Ring<CT, HD, NT>::WARPS * 32, Ring<CT, HD, NT>::CTAS) paged_kernel(const PagedParams p) {
    using R = Ring<CT, HD, NT>;
    constexpr int RB = R::RB, ST = R::STAGES, kWarps = R::WARPS, kBlock = R::BLOCK, HALVES = kBlock / 16;
    constexpr bool I8 = sizeof(CT) == 1, BF = std::is_same<CT, __nv_bfloat16>::value;
    constexpr int KS = HD / 16;        // products along the dims of a score
    constexpr int MT = HD / 16;        // 16-dim tiles of the output
    constexpr int COLS = 8 * NT;
    constexpr int VP = I8 || NT == 1 ? 2 : 1;  // planes of a weight
    // Weights are 2^(LIFT + x) with x <= RISE; at most 2^15 in fp16, where int8 rows' scales take what a LIFT would.
    constexpr int RISE = BF ? 8 : 6, LIFT = BF || I8 ? 0 : 15 - RISE, TOP_SCALE = 15 - RISE;
    // Queries in shared memory where the registers they would take are the warps' that an SM could hold (64 sequences of 5
    // fp32 rows: 41.3 us in registers, 35.4; 64 of 5 fp16 rows, head_dim 128: 81 with two tiles and twice the reading, 60
    // with three).  16-bit ones of two tiles, or at head_dim 64, were 2 to 6% slower so.
    constexpr bool SHARED_Q = NT > 1 && (I8 || (HD == 128 && NT == 3));
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_before, s_seq, s_piece, s_len, s_cuts, s_most, s_last;
    const pf_paged_cache& c = p.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
    const int segs = c.n_kv_heads * p.row_groups;  // of one sequence

    after_previous();
    // ---- this CTA's piece ----  (the host has seen to it that all chunks count in 31 bits)
    if (warp == 0 && p.plan) {
        if (lane == 0) {
            const int4 all = p.plan[0], mine = p.plan[1 + blockIdx.x];  // (there is room for one a CTA)
            s_seq = (int)blockIdx.x < all.x ? mine.x : -1;
            s_piece = mine.y, s_before = mine.z, s_len = mine.w, s_most = all.y;
            s_cuts = cuts_of(chunks_of<R::CHUNK>(mine.w), all.y, 1.0f / (float)all.y);
        }
    } else if (warp == 0) {
        int total = 0;
        bool long_one = false;
        for (int b = lane; b < p.n_seqs; b += 32) {
            const int n = chunks_of<R::CHUNK>(length_of(p, b, blockIdx.x == 0 ? p.err : nullptr));
            total += n;
            long_one |= n > kWhole;
        }
        total = __reduce_add_sync(0xffffffffu, total) * segs;
        const int share = (total + p.ctas - 1) / p.ctas;
        int most = 2 * share;
        if (!__any_sync(0xffffffffu, long_one)) {
            most = kWhole;
        } else if (p.n_seqs * segs < few_segments(p.ctas)) {  // as piece_limit, each lane trying one
            const int mine = share + lane * ((share + 31) / 32);
            const float inv = 1.0f / (float)mine;
            int pieces = 0;
#pragma unroll 4
            for (int b = 0; b < p.n_seqs; b++) pieces += cuts_of(chunks_of<R::CHUNK>(length_of(p, b, nullptr)), mine, inv);
            const unsigned fits = __ballot_sync(0xffffffffu, pieces * segs <= p.ctas);
            most = __shfl_sync(0xffffffffu, mine, fits ? __ffs((int)fits) - 1 : 31);
        }
        const float inv_most = 1.0f / (float)most;
        int pieces = 0, before = 0, found = -1;
        for (int b0 = 0; b0 < p.n_seqs && found < 0; b0 += 32) {
            const int b = b0 + lane, len = b < p.n_seqs ? length_of(p, b, nullptr) : 0;
            const int n = b < p.n_seqs ? chunks_of<R::CHUNK>(len) : 0;
            const int cuts = n ? cuts_of(n, most, inv_most) : 0, my_pieces = cuts * segs, my_chunks = n * segs;
            int upto = my_pieces, upto_chunks = my_chunks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o), y = __shfl_up_sync(0xffffffffu, upto_chunks, o);
                if (lane >= o) upto += x, upto_chunks += y;
            }
            const unsigned here = __ballot_sync(0xffffffffu, (int)blockIdx.x < pieces + upto);
            if (here) {
                const int at = __ffs((int)here) - 1;
                if (lane == at) {
                    s_piece = (int)blockIdx.x - (pieces + upto - my_pieces);
                    s_before = before + upto_chunks - my_chunks;
                    s_len = len;
                    s_cuts = cuts;
                    s_most = most;
                }
                found = b0 + at;
            }
            pieces += __shfl_sync(0xffffffffu, upto, 31);
            before += __shfl_sync(0xffffffffu, upto_chunks, 31);
        }
        if (lane == 0) s_seq = found;
    }
    __syncthreads();
    const int seq = s_seq;
    if (seq < 0) return;  // the grid is an upper bound
    const int len = s_len, chunks = chunks_of<R::CHUNK>(len), cuts = s_cuts, most = s_most;
    const int seg = s_piece / cuts, piece = s_piece - seg * cuts, g = seg / p.row_groups, rg = seg - g * p.row_groups;
    const int seg_begin = s_before + seg * chunks;
    const int ch0 = cuts == 1 ? 0 : (int)((int64_t)chunks * piece / cuts);
    const int ch1 = cuts == 1 ? chunks : (int)((int64_t)chunks * (piece + 1) / cuts);
    const int x0 = rg * COLS, cols = min(COLS, p.cols - x0);  // this row group's columns
    const int sees_all = len - p.rows + 1;                    // entries that the first new token sees

    uint8_t* ring = smem + warp * ST * R::BYTES;
    const uint32_t ring_u32 = (uint32_t)__cvta_generic_to_shared(ring);
    const int64_t page_slots = (int64_t)c.n_layers * c.n_kv_heads * c.page_size;
    // ---- queries, on their way while the ring is set up ----
    // int8: piece j of the row's 16-byte ones that this thread reads is dims 64 j + 16 t ..; 16-bit: 32 j + 8 t ..  With one
    // column tile every warp keeps it in registers; of several each warp prepares its share for all, in shared memory.
    constexpr int MINE = SHARED_Q ? (NT + kWarps - 1) / kWarps : NT;
    float raw[MINE][I8 ? HD / 4 : HD / 8];
#pragma unroll
    for (int y = 0; y < MINE; y++) {
        const int nt = SHARED_Q ? warp + y * kWarps : y, x = 8 * nt + gr;
        const int token = token_of(x0 + x, p.group), head = g * p.group + x0 + x - token * p.group;
        const int64_t at = ((int64_t)seq * p.rows + token) * p.q_stride + head * HD;
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < HD / 64; j++) load16<PLANES>(p.q, at + 64 * j + 16 * t, p.dtype, x < cols, raw[y] + 16 * j);
        } else {
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // bits
                if (x < cols) v = *reinterpret_cast<const float4*>(static_cast<const CT*>(p.q) + at + 32 * j + 8 * t);
                raw[y][4 * j] = v.x, raw[y][4 * j + 1] = v.y, raw[y][4 * j + 2] = v.z, raw[y][4 * j + 3] = v.w;
            }
        }
    }

    // ---- the ring: block k of this warp is entries first(k) .. + 31 ----
    const int n_blocks = ch1 - ch0;
    auto first_entry = [&](int k) { return ((ch0 + k) * kWarps + warp) * kBlock; };
    const int* table = c.table + (int64_t)seq * c.max_pages;
    // The table's entry for the block's 16-entry half (not looked at before the block is asked for: it is on its way);
    // -1: none of the half is there.
    auto page_of = [&](int k, int half) {
        const int e = first_entry(k) + 16 * half;
        return k < n_blocks && e < len ? table[e >> p.page_shift] : -1;
    };
    auto checked = [&](int page, int e) {
        if ((unsigned)page < (unsigned)c.n_pages) return page;
        if (e < len) latch(p.err, ERR_BOUNDS);
        return -1;
    };
    // A half's 16 rows lie behind one another in their page: a pass of 32 lanes is 512 bytes of them, and only its base
    // depends on the block.
    constexpr int PR = RB / 16, STEP = 32 / PR;  // pieces of a row, rows a pass
    const int lane_row = lane / PR, lane_piece = lane % PR;
    const uint32_t key_to = key_at<RB>(lane_row, lane_piece);
    constexpr int VARIANTS = RB == 64 ? 1 : (RB == 128 ? 2 : 4);  // of the values' permutation among passes
    uint32_t value_to[VARIANTS];
#pragma unroll
    for (int i = 0; i < VARIANTS; i++)
        value_to[i] = kBlock * RB + value_at<RB>(i * STEP + lane_row, lane_piece) - i * STEP * RB;
    const int64_t unit_row = ((int64_t)p.layer * c.n_kv_heads + g) * c.page_size;
    auto issue = [&](int k, int page0, int page1) {
        const int e0 = first_entry(k);
        const uint32_t to = ring_u32 + (k % ST) * R::BYTES;
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            const int e = e0 + 16 * half, page = checked(half ? page1 : page0, e);
            const int rows = page < 0 ? 0 : min(len - e, 16);  // of the half's 16; the others are filled with zeros
            const int64_t row = (int64_t)max(page, 0) * page_slots + unit_row + (e & (c.page_size - 1));
            const uint8_t* from_k = static_cast<const uint8_t*>(c.k) + row * RB + lane * 16;
            const uint8_t* from_v = static_cast<const uint8_t*>(c.v) + row * RB + lane * 16;
#pragma unroll
            for (int i = 0; i < 16 / STEP; i++) {
                const int pass = half * (16 / STEP) + i;
                const bool on = i * STEP + lane_row < rows;
                copy16(to + key_to + pass * 512, from_k + i * 512, on);
                copy16(to + value_to[pass % VARIANTS] + pass * 512, from_v + i * 512, on);
            }
            if constexpr (I8) {  // lanes 0-15 the keys' scales, 16-31 the values'
                const float* from = (lane < 16 ? c.k_scale : c.v_scale) + row + (lane & 15);
                copy4(to + 2 * kBlock * RB + (lane < 16 ? 0 : 4 * kBlock) + 64 * half + 4 * (lane & 15), from,
                      (lane & 15) < rows);
            }
        }
    };
    int page0 = page_of(0, 0), page1 = HALVES == 2 ? page_of(0, 1) : -1;
#pragma unroll
    for (int k = 0; k < ST - 1; k++) {
        const int n0 = page_of(k + 1, 0), n1 = HALVES == 2 ? page_of(k + 1, 1) : -1;
        if (k < n_blocks) issue(k, page0, page1);
        copy_commit();
        page0 = n0, page1 = n1;
    }

    // ---- queries into operands ----
    // [plane][product][2]; in shared memory two products' four words are one 16-byte piece a lane
    uint32_t q[SHARED_Q ? 1 : NT][PLANES][KS][2];
    float unit[NT][2];  // score units -> log2 units (log2 e) of this thread's columns 2t, 2t + 1
    uint4* q_shared = reinterpret_cast<uint4*>(smem + R::SMEM);                              // [tile][plane][KS / 2][lane]
    float* unit_shared = reinterpret_cast<float*>(q_shared + NT * PLANES * (KS / 2) * 32);  // [column]
#pragma unroll
    for (int y = 0; y < MINE; y++) {
        const int nt = SHARED_Q ? warp + y * kWarps : y;
        uint32_t(&w)[PLANES][KS][2] = q[SHARED_Q ? 0 : y];
        float all = p.scale * 1.4426950408889634f;
        if constexpr (I8) {
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) big = fmaxf(big, fabsf(raw[y][i]));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const bool finite = big > 0.0f && big < __int_as_float(0x7f800000);
            const int up = finite ? min(13 - exponent_of(big), 100) : 0;  // -114 at least
            const float f = power_of_two(up);
            all *= power_of_two(-up);
#pragma unroll
            for (int i = 0; i < HD / 4; i += 2) {
                const float a = raw[y][i] * f, b = raw[y][i + 1] * f;
                const uint32_t hi = pack<false>(a, b);
                w[0][i / 4][i / 2 % 2] = hi;
                if constexpr (PLANES == 2) {
                    const float2 h = unpack<false>(hi);
                    w[1][i / 4][i / 2 % 2] = pack<false>(a - h.x, b - h.y);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < HD / 8; i++) w[0][i / 2][i % 2] = __float_as_uint(raw[y][i]);
        }
        if constexpr (SHARED_Q) {
            if (nt < NT) {
#pragma unroll
                for (int pl = 0; pl < PLANES; pl++)
#pragma unroll
                    for (int i = 0; i < KS; i += 2)
                        q_shared[((nt * PLANES + pl) * (KS / 2) + i / 2) * 32 + lane] =
                            make_uint4(w[pl][i][0], w[pl][i][1], w[pl][i + 1][0], w[pl][i + 1][1]);
                if (t == 0) unit_shared[8 * nt + gr] = all;
            }
        } else {
            unit[nt][0] = __shfl_sync(0xffffffffu, all, 8 * t);
            unit[nt][1] = __shfl_sync(0xffffffffu, all, 8 * t + 4);
        }
    }
    if constexpr (SHARED_Q) {
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) unit[nt][0] = unit_shared[8 * nt + 2 * t], unit[nt][1] = unit_shared[8 * nt + 2 * t + 1];
    }
    // Entries that this thread's two columns of each tile see.
    int sees[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int x = 8 * nt + 2 * t + i;
            sees[nt][i] = x < cols ? sees_all + token_of(x0 + x, p.group) : 0;
        }

    // ---- running softmax ----
    // LIFT minus the maxima, 0 as long as there is none (`above`, the exponent that calls for a new one, is -inf then).
    float o[MT][NT][4], minus_m[NT][2], above[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        minus_m[nt][0] = minus_m[nt][1] = 0.0f;
        above[nt][0] = above[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; i++) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    }
    float vscale = 1.0f, back = 1.0f;
    for (int k = 0; k < n_blocks; k++) {
        {
            const int n0 = page_of(k + ST, 0), n1 = HALVES == 2 ? page_of(k + ST, 1) : -1;
            __syncwarp();  // every lane is through with the block whose place is filled now
            if (k + ST - 1 < n_blocks) issue(k + ST - 1, page0, page1);
            copy_commit();
            page0 = n0, page1 = n1;
        }
        copy_wait<ST - 1>();
        __syncwarp();
        const int e0 = first_entry(k);
        if (e0 >= len) break;  // the sequence ends in another warp's block
        const uint8_t* kb = ring + (k % ST) * R::BYTES;
        const uint8_t* vb = kb + kBlock * RB;
        const float* scales = reinterpret_cast<const float*>(vb + kBlock * RB);

        // Scores of 16 entries each: rows gr, gr + 8.  All tiles take one product before any takes its next, so that
        // a product does not wait for the one before it.
        float s[HALVES][NT][4];
#pragma unroll
        for (int j = 0; j < RB / 64; j++) {  // pieces t, t + 4, ...
            uint32_t w[HALVES][2][4];
#pragma unroll
            for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 x = *reinterpret_cast<const uint4*>(kb + key_at<RB>(16 * mt + 8 * h + gr, 4 * j + t));
                    w[mt][h][0] = x.x, w[mt][h][1] = x.y, w[mt][h][2] = x.z, w[mt][h][3] = x.w;
                }
#pragma unroll
            for (int i2 = 0; i2 < (I8 ? 4 : 2); i2 += 2) {
                const int k0 = (I8 ? 4 : 2) * j + i2;  // products k0, k0 + 1 along the dims
                uint32_t b[NT][PLANES][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int pl = 0; pl < PLANES; pl++) {
                        if constexpr (SHARED_Q) {
                            const uint4 x = q_shared[((nt * PLANES + pl) * (KS / 2) + k0 / 2) * 32 + lane];
                            b[nt][pl][0] = x.x, b[nt][pl][1] = x.y, b[nt][pl][2] = x.z, b[nt][pl][3] = x.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++) b[nt][pl][e] = q[nt][pl][k0 + e / 2][e % 2];
                        }
                    }
#pragma unroll
                for (int i = i2; i < i2 + 2; i++) {
                    uint32_t f[HALVES][4];
#pragma unroll
                    for (int mt = 0; mt < HALVES; mt++) {
                        if constexpr (I8) {
                            const uint32_t ua = w[mt][0][i] ^ 0x80808080u, ub = w[mt][1][i] ^ 0x80808080u;
                            f[mt][0] = bytes_to_half2(ua, 0x4140), f[mt][2] = bytes_to_half2(ua, 0x4342);
                            f[mt][1] = bytes_to_half2(ub, 0x4140), f[mt][3] = bytes_to_half2(ub, 0x4342);
                        } else {
                            f[mt][0] = w[mt][0][2 * i], f[mt][1] = w[mt][1][2 * i];
                            f[mt][2] = w[mt][0][2 * i + 1], f[mt][3] = w[mt][1][2 * i + 1];
                        }
                    }
#pragma unroll
                    for (int pl = 0; pl < PLANES; pl++)
#pragma unroll
                        for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint32_t b0 = b[nt][pl][2 * (i - i2)], b1 = b[nt][pl][2 * (i - i2) + 1];
                                if (i + j + pl == 0) mma_first<BF>(s[mt][nt], f[mt][0], f[mt][1], f[mt][2], f[mt][3], b0, b1);
                                else mma<BF>(s[mt][nt], f[mt][0], f[mt][1], f[mt][2], f[mt][3], b0, b1);
                            }
                }
            }
        }
        // exponents against the maxima so far; does any lie RISE above?
        const bool tail = e0 + kBlock > sees_all;  // some entry is not seen by every column
        bool rise = false;
        float ks[HALVES][2];
#pragma unroll
        for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) ks[mt][h] = I8 ? scales[16 * mt + 8 * h + gr] : 1.0f;
#pragma unroll
        for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[mt][nt][i] *= unit[nt][i & 1];
        if (tail) {
#pragma unroll
            for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {  // ks may be inf or NaN here: the factor goes in before the mask
                        const bool seen = e0 + 16 * mt + 8 * (i >> 1) + gr < sees[nt][i & 1];
                        s[mt][nt][i] = seen ? s[mt][nt][i] * ks[mt][i >> 1] : -INFINITY;
                    }
#pragma unroll
            for (int mt = 0; mt < HALVES; mt++) ks[mt][0] = ks[mt][1] = 1.0f;
        }
#pragma unroll
        for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // (fma(-inf, 1, 0) where there is no maximum yet)
                    rise |= fmaf(s[mt][nt][i], ks[mt][i >> 1], minus_m[nt][i & 1]) > above[nt][i & 1];
                }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float top = -INFINITY;
#pragma unroll
                    for (int mt = 0; mt < HALVES; mt++)
                        top = fmaxf(top, fmaxf(s[mt][nt][i] * ks[mt][0], s[mt][nt][2 + i] * ks[mt][1]));
#pragma unroll
                    for (int x = 4; x <= 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    // no other column has a say: a row stays the same whatever its neighbours are
                    const bool none = above[nt][i] == -INFINITY;
                    if (none ? top > -INFINITY : top + minus_m[nt][i] > LIFT + RISE) {
                        const float f = none ? 0.0f : exp2_approx(LIFT - minus_m[nt][i] - top);
                        minus_m[nt][i] = LIFT - top;
                        above[nt][i] = LIFT + RISE;
                        l[nt][i] *= f;
                        if (!none)
#pragma unroll
                            for (int d = 0; d < MT; d++) o[d][nt][i] *= f, o[d][nt][2 + i] *= f;
                    }
                }
        }
        // weights
        // int8: 2^up takes the block's largest finite scale to 2^(TOP_SCALE - 1) .., so that p v_scale 2^up < 2^15 (p <= 2^RISE);
        // the one before is kept while it is below 2^TOP_SCALE and not below 2^-7 of that.
        if constexpr (I8) {
            const float inf = __int_as_float(0x7f800000), vs = fabsf(scales[kBlock + lane]), x = vs * vscale;
            constexpr float TOP = 1 << TOP_SCALE, LOW = TOP / 128;
            if (__any_sync(0xffffffffu, x >= TOP && vs < inf) || !__any_sync(0xffffffffu, x >= LOW && x < inf)) {
                const unsigned big = __reduce_max_sync(0xffffffffu, vs < inf ? __float_as_uint(vs) : 0u);
                const int up = min(TOP_SCALE - 1 - exponent_of(__uint_as_float(big)), 100);  // -121 at least
                vscale = power_of_two(up), back = power_of_two(-up);
            }
        }
        uint32_t pw[HALVES][NT][VP][2];  // [entries 16 mt ..][column tile][plane][first, second 8 entries], transposed
#pragma unroll
        for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * mt + 8 * h + gr;
                const float vs = I8 ? scales[kBlock + r] * vscale : 1.0f;
                const bool vs_ok = fabsf(vs) < __int_as_float(0x7f800000);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float y[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float e = exp2_approx(fmaf(s[mt][nt][2 * h + i], ks[mt][h], minus_m[nt][i]));
                        l[nt][i] += e;
                        y[i] = I8 ? e * vs : e;
                        if (I8 && tail && !vs_ok && e0 + r >= sees[nt][i]) y[i] = 0.0f;  // 0 whatever its scale is
                    }
                    if constexpr (I8) {  // (an inf is the largest value and an inf)
                        const uint32_t hi = pack_finite(y[0], y[1]);
                        const float2 got = unpack<false>(hi);
                        pw[mt][nt][0][h] = transpose8x8(hi);
                        pw[mt][nt][1][h] = transpose8x8(pack<false>(y[0] - got.x, y[1] - got.y));
                    } else if constexpr (VP == 2) {
                        // y cut to the type, and what is left of y (1 + 2^-23), which is above 0 (fp16: 2^-24 at least) if y is
                        const uint32_t hi = pack_cut<BF>(y[0], y[1]);
                        const float2 got = unpack<BF>(hi);
                        float lo[2] = {fmaf(y[0], 1.00000012f, -got.x), fmaf(y[1], 1.00000012f, -got.y)};
                        if constexpr (!BF) lo[0] = fmaxf(lo[0], fminf(y[0], 0x1p-24f)), lo[1] = fmaxf(lo[1], fminf(y[1], 0x1p-24f));
                        pw[mt][nt][0][h] = transpose8x8(hi);
                        pw[mt][nt][1][h] = transpose8x8(pack<BF>(lo[0], lo[1]));
                    } else {
                        pw[mt][nt][0][h] = transpose8x8(pack<BF>(y[0], y[1]));
                    }
                }
            }
        // values
        const int passes = !I8 && tail && p.rows > 1 ? p.rows : 1;
        for (int pass = 0; pass < passes; pass++) {
            // one pass for all, or one a new token with what it may not see set to 0
            const int upto = passes == 1 ? INT_MAX : sees_all + pass - e0;
            constexpr int VB = RB == 64 ? 8 : 16;  // bytes of a row this thread reads at a time
            constexpr int W = VB / 4, GROUPS = RB / 8 / VB, PER = MT / GROUPS;
#pragma unroll
            for (int gi = 0; gi < GROUPS; gi++) {
                uint32_t v[HALVES][4][W];  // entries 16 mt + 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int mt = 0; mt < HALVES; mt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 16 * mt + 2 * t + (e & 1) + 8 * (e >> 1);
                        if constexpr (W == 2) {
                            const uint2 x = *reinterpret_cast<const uint2*>(vb + value_at<RB>(r, gr >> 1) + 8 * (gr & 1));
                            v[mt][e][0] = x.x ^ 0x80808080u, v[mt][e][1] = x.y ^ 0x80808080u;
                        } else {
                            uint4 x = *reinterpret_cast<const uint4*>(vb + value_at<RB>(r, 8 * gi + gr));
                            if (!I8 && r >= upto) x = make_uint4(0, 0, 0, 0);
                            const uint32_t flip = I8 ? 0x80808080u : 0u;
                            v[mt][e][0] = x.x ^ flip, v[mt][e][1] = x.y ^ flip, v[mt][e][2] = x.z ^ flip, v[mt][e][3] = x.w ^ flip;
                        }
                    }
#pragma unroll
                for (int i = 0; i < PER; i += 2) {  // two dim tiles at once, for the same reason
                    float acc[2][NT][4];
#pragma unroll
                    for (int mt = 0; mt < HALVES; mt++) {
                        uint32_t f[2][4];
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            if constexpr (I8) {
                                // word i / 2: four dims; its first two or last two, of two entries each
                                const uint32_t sel = y ? 0x7362 : 0x5140;
                                const uint32_t a = __byte_perm(v[mt][0][i / 2], v[mt][1][i / 2], sel);
                                const uint32_t b = __byte_perm(v[mt][2][i / 2], v[mt][3][i / 2], sel);
                                f[y][0] = bytes_to_half2(a, 0x4140), f[y][1] = bytes_to_half2(a, 0x4342);
                                f[y][2] = bytes_to_half2(b, 0x4140), f[y][3] = bytes_to_half2(b, 0x4342);
                            } else {
                                f[y][0] = __byte_perm(v[mt][0][i + y], v[mt][1][i + y], 0x5410);
                                f[y][1] = __byte_perm(v[mt][0][i + y], v[mt][1][i + y], 0x7632);
                                f[y][2] = __byte_perm(v[mt][2][i + y], v[mt][3][i + y], 0x5410);
                                f[y][3] = __byte_perm(v[mt][2][i + y], v[mt][3][i + y], 0x7632);
                            }
                        }
#pragma unroll
                        for (int pl = 0; pl < VP; pl++)
#pragma unroll
                            for (int y = 0; y < 2; y++)
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    const uint32_t b0 = pw[mt][nt][pl][0], b1 = pw[mt][nt][pl][1];
                                    if (mt + pl == 0) mma_first<BF>(acc[y][nt], f[y][0], f[y][1], f[y][2], f[y][3], b0, b1);
                                    else mma<BF>(acc[y][nt], f[y][0], f[y][1], f[y][2], f[y][3], b0, b1);
                                }
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if (!I8 && passes > 1 && sees[nt][e & 1] != upto + e0) continue;  // another token's pass
                                float& to = o[gi * PER + i + y][nt][e];
                                to = I8 ? fmaf(acc[y][nt][e], back, to) : to + acc[y][nt][e];
                            }
                }
            }
        }
    }
    copy_wait<0>();

    // ---- the warps' shares together ----
    // smem: [warp][column][HD + 2], a row's last two its maximum and sum
    constexpr int PITCH = HD + 2, PART = HD + 4;  // here, and in `part` (16-byte loads)
    float* shared = reinterpret_cast<float*>(smem);
    static_assert(kWarps * COLS * PITCH * 4 <= R::SMEM && COLS * kMaxCuts * 4 <= R::SMEM, "the shares fit the ring");
    __syncthreads();  // the rings are empty
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float sum = l[nt][i];
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            float* to = shared + (warp * COLS + 8 * nt + 2 * t + i) * PITCH;
            if (gr == 0) to[HD] = above[nt][i] == -INFINITY ? -INFINITY : -minus_m[nt][i], to[HD + 1] = sum;
#pragma unroll
            for (int d = 0; d < MT; d++) {
                // tile d's rows gr and gr + 8 are two neighbouring dims
                constexpr int VB = RB == 64 ? 8 : 16, PER = MT / (RB / 8 / VB), DIMS = VB / (int)sizeof(CT);
                const int dim = d / PER * (HD / (MT / PER)) + gr * DIMS + 2 * (d % PER);
                *reinterpret_cast<float2*>(to + dim) = make_float2(o[d][nt][i], o[d][nt][2 + i]);
            }
        }
    __syncthreads();
    // A cut segment is longer than P = `most` chunks, so no two have one seg_begin / P, and its pieces fit twice that
    // many places.
    const int place = seg_begin / most;
    float* part = p.part + (int64_t)(2 * place + piece) * COLS * PART;
    if (threadIdx.x < cols) {  // a column's factors, in the place of the warps' maxima
        float* at = shared + threadIdx.x * PITCH + HD;
        float top = -INFINITY, sum = 0.0f, f[kWarps];
#pragma unroll
        for (int s = 0; s < kWarps; s++) top = fmaxf(top, at[s * COLS * PITCH]);
#pragma unroll
        for (int s = 0; s < kWarps; s++) {
            const float m = at[s * COLS * PITCH];
            f[s] = m == -INFINITY ? 1.0f : exp2_approx(m - top);  // no maximum: its shares are zeros, or NaN
            sum += at[s * COLS * PITCH + 1] * f[s];
        }
        if (cuts > 1) __stcg(reinterpret_cast<float2*>(part + threadIdx.x * PART + HD), make_float2(top, sum));
        const float inv = cuts > 1 ? 1.0f : (sum == 0.0f ? 0.0f : 1.0f / sum);
#pragma unroll
        for (int s = 0; s < kWarps; s++) at[s * COLS * PITCH] = f[s] * inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cols * (HD / 2); i += kWarps * 32) {
        const int x = i / (HD / 2), d = i % (HD / 2) * 2;
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < kWarps; s++) {
            const float* from = shared + (s * COLS + x) * PITCH;
            const float2 y = *reinterpret_cast<const float2*>(from + d);
            v.x += y.x * from[HD], v.y += y.y * from[HD];
        }
        if (cuts == 1) store_out(p, seq, g, x0 + x, d, HD, v);
        else __stcg(reinterpret_cast<float2*>(part + x * PART + d), v);
    }
    if (cuts > 1) {
        // ---- the segment's pieces together, by the last to come ----
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicAdd(&p.count[place], 1) == cuts - 1;
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (threadIdx.x == 0) p.count[place] = 0;  // as it was found
        const float* parts = p.part + (int64_t)2 * place * COLS * PART;
        float* factor = shared;  // [column][kMaxCuts]
        for (int x = warp; x < cols; x += kWarps) {  // two pieces a lane
            float2 ms[2];
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int k = lane + 32 * i;
                ms[i] = k < cuts ? __ldcg(reinterpret_cast<const float2*>(parts + ((int64_t)k * COLS + x) * PART + HD))
                                 : make_float2(-INFINITY, 0.0f);
                top = fmaxf(top, ms[i].x);
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
            for (int i = 0; i < 2; i++) {
                ms[i].x = ms[i].x == -INFINITY ? 1.0f : exp2_approx(ms[i].x - top);
                sum += ms[i].y * ms[i].x;
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int i = 0; i < 2; i++) factor[x * kMaxCuts + lane + 32 * i] = ms[i].x * inv;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < cols * (HD / 4); i += kWarps * 32) {
            const int x = i / (HD / 4), d = i % (HD / 4) * 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
            for (int k = 0; k < cuts; k++) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(parts + ((int64_t)k * COLS + x) * PART + d));
                const float f = factor[x * kMaxCuts + k];
                v.x += y.x * f, v.y += y.y * f, v.z += y.z * f, v.w += y.w * f;
            }
            store_out(p, seq, g, x0 + x, d, HD, make_float2(v.x, v.y));
            store_out(p, seq, g, x0 + x, d + 2, HD, make_float2(v.z, v.w));
        }
    }
}

// Column tiles of 8 that a CTA takes: the rows' in as few equal groups as the registers allow, as each group reads the cache
// anew.  (Four tiles or two groups of two, head_dim 64, 64 sequences of 7,000 to 8,000 entries: bf16 208 and 286 us, int8 with
// fp16 rows 272 and 295, with fp32 rows 310 and 317.  Short contexts of int8 rows, where four tiles spill and the half as many
// segments are cut, lose by it: 512 to 1,024 entries of 4 kv heads 41 and 27 us; of 8 kv heads 48 and 46.)
int tiles_for(int cols, int head_dim) {
    const int tiles = ceil_div(cols, 8), groups = ceil_div(tiles, head_dim == 64 ? 4 : 3);
    return ceil_div(tiles, groups);
}

int cta_limit(const pf_paged_cache& c, int tiles) {
    return 148 * ctas_per_sm(c.head_dim * type_bytes(c.dtype), c.dtype == PF_I8, tiles);
}

// Of `work`: the counters, the pieces of cut segments, the plan.
size_t part_bytes(const pf_paged_cache& c, int tiles) {
    return (size_t)(cta_limit(c, tiles) + 1) * 2 * 8 * tiles * (c.head_dim + 4) * sizeof(float);
}

size_t plan_bytes(const pf_paged_cache& c, int tiles, int n_seqs, int cols) {
    const size_t segments = (size_t)n_seqs * c.n_kv_heads * ceil_div(cols, 8 * tiles);
    return (1 + segments + cta_limit(c, tiles)) * sizeof(int4);
}

template <typename CT, int HD, int NT, int PLANES>
pf_status launch_tiles(PagedParams& p, cudaStream_t st) {
    using R = Ring<CT, HD, NT>;
    p.row_groups = ceil_div(p.cols, 8 * NT);
    p.ctas = cta_limit(p.c, NT);
    // segments, and with pieces of total / CTAs chunks or more no more than that many cuts
    const int64_t segments = (int64_t)p.n_seqs * p.c.n_kv_heads * p.row_groups;
    const int64_t chunks = std::max<int64_t>(((int64_t)p.c.max_pages * p.c.page_size + R::CHUNK - 1) / R::CHUNK, 1);
    const int64_t grid = std::min(segments * chunks, segments + p.ctas);
    PF_CHECK(2 * segments * chunks <= INT32_MAX, "pf_paged_attention: too many positions for one call");
    if (p.n_seqs >= (segments < few_segments(p.ctas) ? kPlannedFew : kPlanned))
        p.plan = reinterpret_cast<int4*>(reinterpret_cast<char*>(p.part) + part_bytes(p.c, NT));
    constexpr int SMEM = R::SMEM + (NT > 1 ? NT * PLANES * (HD / 32) * 512 + 8 * NT * 4 : 0);  // the ring; queries, where they are shared
    if (p.plan) PF_TRY(launch_after("paged_attention_plan", plan_kernel, dim3(1), kDecide, 0, st, p, R::CHUNK));
    static std::atomic<uint64_t> attr{0};
    PF_TRY(raise_smem_limit(paged_kernel<CT, HD, NT, PLANES>, SMEM, attr));
    return launch_after("paged_attention", paged_kernel<CT, HD, NT, PLANES>, dim3((unsigned)grid), R::WARPS * 32, SMEM, st, p);
}

template <typename CT, int PLANES>
pf_status launch_paged(PagedParams& p, cudaStream_t st) {
    const int nt = tiles_for(p.cols, p.c.head_dim);
    if (p.c.head_dim == 128) {
        if (nt == 1) return launch_tiles<CT, 128, 1, PLANES>(p, st);
        return nt == 2 ? launch_tiles<CT, 128, 2, PLANES>(p, st) : launch_tiles<CT, 128, 3, PLANES>(p, st);
    }
    if (nt == 1) return launch_tiles<CT, 64, 1, PLANES>(p, st);
    if (nt == 2) return launch_tiles<CT, 64, 2, PLANES>(p, st);
    return nt == 3 ? launch_tiles<CT, 64, 3, PLANES>(p, st) : launch_tiles<CT, 64, 4, PLANES>(p, st);
}

}  // namespace

}  // namespace pf

using namespace pf;

extern "C" {

size_t pf_paged_attention_work_bytes(const pf_paged_cache* c, int32_t n_seqs, int32_t rows, int32_t n_heads) {
    if (check_paged_sizes(c, "pf_paged_attention_work_bytes") != PF_OK || n_seqs < 0 || n_seqs > 1 << 20 || rows < 1 || rows > 8 ||
        n_heads < 1 || n_heads > kMaxHeads || n_heads % c->n_kv_heads)
        return 0;
    const int nt = tiles_for(n_heads / c->n_kv_heads * rows, c->head_dim);
    return kCounters * sizeof(int) + part_bytes(*c, nt) + (n_seqs < kPlannedFew ? 0 : plan_bytes(*c, nt, n_seqs, n_heads / c->n_kv_heads * rows));
}

pf_status pf_paged_attention(const pf_paged_cache* c, int32_t layer, const void* q, int64_t q_stride, void* out,
                             int64_t out_stride, int32_t dtype, int32_t n_seqs, int32_t rows, int32_t n_heads,
                             float scale, void* work, size_t work_bytes, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_attention", false));
    PF_CHECK(layer >= 0 && layer < c->n_layers, "pf_paged_attention: layer %d of %d", layer, c->n_layers);
    PF_CHECK(n_seqs >= 0 && n_seqs <= c->max_seqs, "pf_paged_attention: %d sequences of %d", n_seqs, c->max_seqs);
    PF_CHECK(rows >= 1 && rows <= 8, "pf_paged_attention: %d rows are not 1 to 8", rows);
    PF_CHECK(n_heads > 0 && n_heads <= kMaxHeads && n_heads % c->n_kv_heads == 0,
             "pf_paged_attention: %d heads over %d kv heads", n_heads, c->n_kv_heads);
    PF_CHECK(c->dtype == PF_I8 ? dtype == PF_F32 || dtype == PF_BF16 || dtype == PF_F16 : dtype == c->dtype,
             "pf_paged_attention: rows of dtype %d over a cache of dtype %d", dtype, c->dtype);
    PF_CHECK(scale > 0.0f && scale <= kMaxScale, "pf_paged_attention: scale must be positive and at most 2.3e38");
    const int64_t width = (int64_t)n_heads * c->head_dim, es = type_bytes(dtype);
    PF_CHECK(q_stride >= width && out_stride >= width && q_stride * es % 16 == 0 && out_stride * es % 16 == 0 &&
                 (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0,
             "pf_paged_attention: rows are narrower than the heads or not 16-byte aligned");
    const size_t need = pf_paged_attention_work_bytes(c, n_seqs, rows, n_heads);
    PF_CHECK(work_bytes >= need && (uintptr_t)work % 16 == 0, "pf_paged_attention: work of %zu bytes, %zu needed",
             work_bytes, need);
    PF_TRY(require_device());
    if (n_seqs == 0) return PF_OK;
    PF_CHECK(q && out && work, "pf_paged_attention: null argument");
    PagedParams p{};
    p.c = *c, p.q = q, p.out = out, p.q_stride = q_stride, p.out_stride = out_stride;
    p.layer = layer, p.n_seqs = n_seqs, p.rows = rows, p.n_heads = n_heads, p.dtype = dtype;
    p.group = n_heads / c->n_kv_heads, p.cols = p.group * rows;
    p.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    p.scale = scale;
    p.count = static_cast<int*>(work);
    p.part = reinterpret_cast<float*>(static_cast<char*>(work) + kCounters * sizeof(int));
    p.err = device_error_flag();
    cudaStream_t st = as_stream(stream);
    if (c->dtype == PF_BF16) return launch_paged<__nv_bfloat16, 1>(p, st);
    if (c->dtype == PF_F16) return launch_paged<__half, 1>(p, st);
    return dtype == PF_F32 ? launch_paged<int8_t, 2>(p, st) : launch_paged<int8_t, 1>(p, st);
}

}  // extern "C"
