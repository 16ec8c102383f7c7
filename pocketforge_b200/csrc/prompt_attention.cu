// prompt_attention.cu — causal attention over packed prompts on the
// 5th-generation tensor cores.
//
//   out_i = sum_{j <= i} softmax_j(scale * q_i . k_j) v_j   within a sequence
//
// in one pass over the keys: blocks of 128, the running row maximum m and sum
// l in fp32, out = O / l at the end.
//
// A query tile's 128 rows are F heads of one kv head at 128 / F tokens, F the
// largest power of two in the group (up to 32): short sequences and the ends of
// long ones fill tiles that 128 tokens of one head would leave mostly empty.  A
// work unit is two such tiles of one kv head; every K and V block is loaded once
// for both.  One CTA an SM takes unit after unit (clusterlaunchcontrol: a running
// CTA takes over the launch of the next one, so the units go to whoever is
// free, longest first within a sequence).  Its warps:
//   0-3, 4-7  softmax of tile 0 and 1, one row a thread: scores from TMEM,
//             p = 2^(c s - c m) (c = scale log2 e), p as 16-bit back into TMEM,
//             at the end O / l to memory
//   8         unit list and TMA loads, one lane a 64-column slab
//   9         issues the tcgen05 products S = Q K^T and O += P V
//   10        looks through the V block on the diagonal (below)
// The blocks of all its units are one stream of products.  At head_dim 64 the
// scores of the next block (or unit) are computed while this block's are
// exponentiated; at 128 TMEM has no room for that, P overlays the scores it came
// from and the two tiles take turns at the tensor cores.
//
// What bounds it (B200, measured): 8,192 tokens, 32 heads over 8, head_dim 128,
// bf16: 550 GFLOP in 500 us, 1.10 PFLOP/s, 79% of what cuBLAS sustains under the
// power cap (ncu: tensor pipe and special-function unit are each active in 64% of
// the cycles at 1.6 GHz; the two tiles wait for both in turn, and the clock is
// the power cap's).  64 prompts of 33 to 1,024 tokens, head_dim 64: 151 us (163
// with one head a tile; 256 prompts of 5 to 40 tokens, 8 heads a kv head: 80 and
// 235; 8,192 tokens: 500 and 496); half of the products are in blocks on the
// diagonal or behind the end, the special-function unit takes 2,048 of a full
// block's 3,100 cycles, and each unit of three blocks on average has about 4,000
// cycles of its own (first scores, output): 280,000 cycles for an SM's 63 blocks
// and 21 units, where 267,000 are counted (special-function unit active in 41% of
// them, tensor pipe in 23%).
// Short units run every path of the code once, so its size counts: 84 KB of
// unrolled code ran 221 us where 60 KB ran 174 (stalls for instructions 1.9 an
// issue before, 0.2 after).  Measured and not kept: a part of the exponentials by
// a polynomial on the FMA pipe (498 to 509 us on 8,192 tokens), two threads a row
// (550), exponents against the last block's maximum while this one's is found
// (524), turns at the special-function unit (515).
//
// The maximum that the exponents refer to rises only when a block exceeds it
// by 2^8 (fp16: 2^6), so O (in TMEM) is rescaled rarely, and the row sum takes the
// same p.
//
// Rounding: scores, maxima, sums and O are fp32.  P is rounded to the inputs'
// 16-bit type, which the tensor core asks for (both operands of one type).  fp16
// ends at 2^-24, and a long row's many p below that can be its answer where the
// largest ones meet small values: p is taken 2^9 times, so that the largest are at
// the end of fp16's range (2^15), and is off by 2^-34 of the row's largest at most
// beside its rounding.
//
// What a row must not see: scores behind the row itself are -inf, their p is 0.
// But 0 x inf = NaN, so V rows behind the sequence's end (another sequence's)
// are set to 0 in shared memory, and so is each inf or NaN among the V rows of
// a block on the diagonal.  The rows that see one have it added to their output
// again: every weight is positive, so inf x p is inf whatever p is.  That is a
// walk over at most 256 keys a row, however long the prompt is.  (One walk for all
// of a warp's rows came out of the compiler with a block's loop 3% slower.)
//
// Every wait is bounded (about a second): a timeout latches ERR_TIMEOUT, the
// other roles stop waiting, and the CTA lets its copies land and frees its TMEM.
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged.cuh"

namespace pf {

namespace {

constexpr int BM = 128;            // query rows a tile, keys a block
constexpr int kSoftmaxWarps = 8;
constexpr int kThreads = 384;      // three warpgroups, the last warp idle
// Registers: the launch gives every thread 168 (64,512 in all).  The softmax
// warpgroups hold a row of 128 scores and take 200 once the third one has gone
// down to 104: 2 x 128 x 200 + 128 x 104 = 64,512.
constexpr int kRegsSoftmax = 200, kRegsOther = 104;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= 384 * 168, "register split");
constexpr uint32_t ERR_TIMEOUT = 16u;
constexpr int kSlots = 2;          // units in the list between the load warp and the others

struct PromptParams {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int* offsets;
    int n_seqs, n_tokens, n_heads, n_kv_heads;
    int pack, packs;  // a tile holds 1 << pack heads; packs of them make the heads of a kv head
    float scale;
    uint32_t* err;
};

template <int HD>
struct Layout {
    static constexpr int NC = HD / 64;                // 64-column (128-byte) slabs of a row
    static constexpr int SLAB = BM * 128;             // bytes of one
    static constexpr int TILE = NC * SLAB;            // a Q tile, K block or V block
    static constexpr int STAGES = HD == 64 ? 4 : 2;   // K blocks and V blocks in flight
    static constexpr int QB = HD == 64 ? 2 : 1;       // buffers of each Q tile: the next unit's, where there is room
    static constexpr int K_OFF = 2 * QB * TILE, V_OFF = K_OFF + STAGES * TILE;
    static constexpr int OUT_OFF = V_OFF + STAGES * TILE;  // 32 rows x 128 bytes of output a softmax warp
    static constexpr int BAR_OFF = OUT_OFF + kSoftmaxWarps * 32 * 128;
    static constexpr int SMEM = BAR_OFF + 512 + 1024;  // barriers, unit list; alignment
    // TMEM columns.  head_dim 64: P has its own columns, so the next scores are
    // computed while this block's are exponentiated; at 128 the accumulators
    // take that room and P overlays the scores it came from.
    static constexpr bool OWN_P = HD == 64;
    static constexpr uint32_t S = 0, P = OWN_P ? 256 : 0, P_STEP = OWN_P ? 64 : 128, O = OWN_P ? 384 : 256;
};

// ---- PTX ----
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Predicated, not branched around: the code on both sides stays one block to schedule.
__device__ __forceinline__ void mbar_arrive_if(uint32_t bar, bool on) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
        "r"((int)on)
        : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Sleeps in hardware for up to the hint's 10 ms (a short default would have the waiting warps poll the issue slots away).
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(10000000u)
        : "memory");
    return ok != 0;
}
// False when a second has passed, or another role has given up.
__device__ __forceinline__ bool mbar_spin(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    uint64_t t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
#pragma unroll 1
    do {
        if (mbar_try_wait(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    } while (!*abort_flag && t - t0 < 1000000000ull);
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return mbar_try_wait(bar, parity) || mbar_spin(bar, parity, abort_flag);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// Operand descriptors, 128-byte swizzle (8 rows of 128 bytes = one 1,024-byte
// atom), version 1 (sm_100), layout type 2.  K-major (Q, K): atoms 1,024 bytes
// apart along the rows.  Rows-as-K (V): 64 columns an atom, the next 64 a slab
// away (leading offset), the next 8 rows 1,024 bytes away (stride offset).
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D fp32; A and B fp16 (0) or bf16 (1); B's major at bit 16; N >> 3; M >> 4.
__host__ __device__ constexpr uint32_t idesc_f16(int bf16, int n, int b_rows_as_k) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_rows_as_k << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// One lane of a warp that is all here.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 in one register pair (one instruction for both on sm_100).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Largest of r[0 .. N).
template <int N>
__device__ __forceinline__ float row_max(const uint32_t* r) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int q = 0; q < N; q += 8)
#pragma unroll
        for (int w = 0; w < 4; w++)
            mx[w] = fmaxf(fmaxf(mx[w], __uint_as_float(r[q + w])), __uint_as_float(r[q + 4 + w]));
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// 16 pairs of scores to p = 2^(c s + off), rounded and packed; sum takes the unrounded ones.  All on the
// special-function unit.
template <typename T>
__device__ __forceinline__ void exponentials(const uint32_t* r, float c, float off, float2 (&sum)[2], uint32_t* pk) {
#pragma unroll
    for (int q = 0; q < 16; q++) {
        float2 x = fma2(make_float2(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1])), make_float2(c, c),
                        make_float2(off, off));
        x.x = ex2(x.x);
        x.y = ex2(x.y);
        sum[q & 1] = add2(sum[q & 1], x);
        pk[q] = pack2<T>(x.x, x.y);
    }
}

// ---- units ----
struct Unit {
    int first, len;   // the sequence's first row and rows
    int g;            // kv head
    int last[2];      // of query tile s: last key block (the one on the diagonal), -1: no such tile
    int token[2];     // first token
    int head[2];      // first head
    int bad;          // an inf or NaN in a V block on the diagonal
    __device__ int blocks() const { return max(last[0], last[1]) + 1; }
};

// Walks the sequences to unit u; a whole warp, the same in every lane.  Each
// lane keeps one sequence of a window of 32, so the offsets are read once a window.
struct UnitList {
    int seq = 0;               // first sequence of the window
    long long before = 0;      // units before it
    long long first_unit = 0, end_unit = -1;  // this lane's sequence, from the window's beginning; -1: not read yet
    int first = 0, len = 0, pairs = 0;
    __device__ bool find(const PromptParams& p, long long u, Unit& out) {
        if (u < before) seq = 0, before = 0, end_unit = -1;
        const int lane = threadIdx.x & 31, tokens = BM >> p.pack;
        while (seq < p.n_seqs) {
            if (end_unit < 0) {
                first = len = 0;
                if (seq + lane < p.n_seqs) {
                    first = p.offsets[seq + lane];
                    const int end = p.offsets[seq + lane + 1];
                    if (first >= 0 && end >= first && end <= p.n_tokens) len = end - first;
                    else latch(p.err, ERR_BOUNDS);
                }
                // a bad list's sequences may overlap: 64 bits, though a good one's units fit 31
                const long long two = ((long long)((len + tokens - 1) >> (7 - p.pack)) * p.packs + 1) / 2;
                pairs = (int)min(two, 0x7fffffffll);
                end_unit = two * p.n_kv_heads;
                first_unit = end_unit;
#pragma unroll 1
                for (int o = 1; o < 32; o <<= 1) {
                    const long long x = __shfl_up_sync(0xffffffffu, end_unit, o);
                    if (lane >= o) end_unit += x;
                }
                first_unit = end_unit - first_unit;
            }
            const unsigned here = __ballot_sync(0xffffffffu, u < before + end_unit);
            if (here) {
                const int at = __ffs((int)here) - 1;
                const int r = (int)(u - before - __shfl_sync(0xffffffffu, first_unit, at));
                out.first = __shfl_sync(0xffffffffu, first, at);
                out.len = __shfl_sync(0xffffffffu, len, at);
                const int q = r / p.n_kv_heads, c = 2 * (__shfl_sync(0xffffffffu, pairs, at) - 1 - q);
                out.g = r - q * p.n_kv_heads;
                // tiles c and c + 1 of (tokens, heads), heads fastest
                const int t = c / p.packs, h = c - t * p.packs, wraps = h + 1 == p.packs;
                out.token[0] = t * tokens, out.token[1] = (t + wraps) * tokens;
                out.last[0] = out.token[0] / BM, out.last[1] = out.token[1] < out.len ? out.token[1] / BM : -1;
                out.head[0] = (out.g * p.packs + h) << p.pack;
                out.head[1] = (out.g * p.packs + (wraps ? 0 : h + 1)) << p.pack;
                return true;
            }
            before += __shfl_sync(0xffffffffu, end_unit, 31);
            seq += 32;
            end_unit = -1;
        }
        return false;
    }
};

// Adds to a row's output the inf and NaN among the values of its tile's first block and the one before it, as far as the row
// sees them: those that the guard has set to 0, and maybe some that are in the output already, which changes nothing.
template <typename T, int HD>
__device__ __noinline__ void add_nonfinite(const PromptParams& p, int first, int token, int head, int g, int token0) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31;
    float sum[N];
#pragma unroll
    for (int d = 0; d < N; d++) sum[d] = 0.0f;
#pragma unroll 4
    for (int key = max(token0 / BM - 1, 0) * BM; key <= token; key++)
#pragma unroll
        for (int d = 0; d < N; d++) {
            const float v = (float)static_cast<const T*>(p.v)[((int64_t)first + key) * p.v_stride + g * HD + lane + 32 * d];
            if (!(fabsf(v) <= 3.402823466e38f)) sum[d] += v;
        }
    T* out = static_cast<T*>(p.out) + ((int64_t)first + token) * p.out_stride + head * HD + lane;
#pragma unroll
    for (int d = 0; d < N; d++)
        if (sum[d] != 0.0f) out[32 * d] = (T)((float)out[32 * d] + sum[d]);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
    using Ly = Layout<HD>;
    constexpr int ST = Ly::STAGES, NC = Ly::NC;
    constexpr int BF = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    const uint32_t bars = base + Ly::BAR_OFF;
    constexpr int QB = Ly::QB;
    auto s_full = [&](int s) { return bars + 8u * (0 + s); };
    auto s_free = [&](int s) { return bars + 8u * (2 + s); };
    auto p_half = [&](int s) { return bars + 8u * (4 + s); };  // p of the block's first 64 keys
    auto p_full = [&](int s) { return bars + 8u * (6 + s); };
    auto o_full = [&](int s) { return bars + 8u * (8 + s); };
    auto o_free = [&](int s) { return bars + 8u * (10 + s); };
    auto u_full = [&](int i) { return bars + 8u * (12 + i); };
    auto u_empty = [&](int i) { return bars + 8u * (14 + i); };
    auto u_seen = [&](int i) { return bars + 8u * (16 + i); };  // the guard is through with the unit
    const uint32_t next_full = bars + 8u * 18;
    auto q_full = [&](int s, uint32_t use) { return bars + 8u * (19 + s * QB + use % QB); };
    auto q_empty = [&](int s, uint32_t use) { return bars + 8u * (19 + 2 * QB + s * QB + use % QB); };
    auto k_full = [&](int i) { return bars + 8u * (19 + 4 * QB + i); };
    auto k_empty = [&](int i) { return bars + 8u * (19 + 4 * QB + ST + i); };
    auto v_full = [&](int i) { return bars + 8u * (19 + 4 * QB + 2 * ST + i); };
    auto v_empty = [&](int i) { return bars + 8u * (19 + 4 * QB + 3 * ST + i); };
    auto v_good = [&](int i) { return bars + 8u * (19 + 4 * QB + 4 * ST + i); };  // looked through
    auto q_tile = [&](int s, uint32_t use) { return base + (uint32_t)((s * QB + use % QB) * Ly::TILE); };
    static_assert(8 * (19 + 4 * QB + 5 * ST) <= 384, "barriers");
    uint8_t* tail = smem + Ly::BAR_OFF + 384;
    const uint32_t next_at = base + Ly::BAR_OFF + 384;                   // 16 bytes: the next unit's launch
    volatile Unit* units = reinterpret_cast<volatile Unit*>(tail + 16);  // [kSlots]
    static_assert(16 + kSlots * sizeof(Unit) + 12 <= 128, "unit list");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 16 + kSlots * sizeof(Unit));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* any = reinterpret_cast<int*>(tmem_slot + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    UnitList list;
    Unit unit;
    after_previous();
    if (warp == 8) {
        const bool found = list.find(p, blockIdx.x, unit);
        if (lane == 0) {
            *any = found;
            for (int s = 0; s < 2; s++) {
                for (int i = 0; i < QB; i++) {
                    mbar_init(q_full(s, i), NC);
                    mbar_init(q_empty(s, i), 1);
                }
                mbar_init(s_full(s), 1);
                mbar_init(s_free(s), 4);
                mbar_init(p_half(s), 4);
                mbar_init(p_full(s), 4);
                mbar_init(o_full(s), 1);
                mbar_init(o_free(s), 4);
            }
            for (int i = 0; i < kSlots; i++) {
                mbar_init(u_full(i), 1);
                mbar_init(u_empty(i), kSoftmaxWarps + 2);
                mbar_init(u_seen(i), 1);
            }
            mbar_init(next_full, 1);
            for (int i = 0; i < ST; i++) {
                mbar_init(k_full(i), NC);
                mbar_init(k_empty(i), 1);
                mbar_init(v_full(i), NC);
                mbar_init(v_empty(i), 2);
                mbar_init(v_good(i), 1);
            }
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    __syncthreads();
    if (!*any) return;  // the grid is an upper bound of the units
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag); };
    auto give_up = [&]() {  // a wait ran out, here or (again) elsewhere
        *abort_flag = 1;
        latch(p.err, ERR_TIMEOUT);
    };
    // The unit in the list's slot, as the load warp left it.
    auto take = [&](int i, Unit& u) {
        volatile Unit& v = units[i];
        u.first = v.first, u.len = v.len, u.g = v.g, u.last[0] = v.last[0], u.last[1] = v.last[1];
    };

    if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 8) {
        // ---------------- unit list, loads ----------------
        // Lane roles: K slabs, V slabs, then Q tile 0's and 1's slabs.  Copies issued by one lane complete one
        // after another, hence a lane for each.
        const int role = lane / NC, c = lane % NC;
        uint32_t it = 0, taken[2] = {0, 0}, last_bar = 0, last_parity = 0;
        bool more = true, ok = true;
        uint32_t n = 0;
        for (;; n++) {
            const int slot = n % kSlots;
            if (lane == 0) {
                ok = wait(u_empty(slot), ((n / kSlots) & 1) ^ 1);
                if (ok) {
                    volatile Unit& v = units[slot];
                    v.first = unit.first, v.len = more ? unit.len : 0, v.g = unit.g;
                    v.last[0] = unit.last[0], v.last[1] = unit.last[1], v.token[0] = unit.token[0], v.token[1] = unit.token[1];
                    v.head[0] = unit.head[0], v.head[1] = unit.head[1];
                    v.bad = 0;
                    mbar_arrive(u_full(slot));
                }
                if (ok && more) {  // ask for the next one
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_expect_tx(next_full, 16);
                    asm volatile(
                        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::
                            "r"(next_at), "r"(next_full)
                        : "memory");
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            if (!ok || !more) break;
            const int nb = unit.blocks();
            if (role < 2) {
                const CUtensorMap* map = role == 0 ? &map_k : &map_v;
                const uint32_t tiles = base + (role == 0 ? Ly::K_OFF : Ly::V_OFF) + c * Ly::SLAB;
#pragma unroll 1
                for (int j = 0; j < nb && ok; j++) {
                    const uint32_t i = it + j, st = i % ST;
                    const uint32_t full = role == 0 ? k_full(st) : v_full(st);
                    ok = wait(role == 0 ? k_empty(st) : v_empty(st), ((i / ST) & 1) ^ 1);
                    if (!ok) break;
                    mbar_expect_tx(full, Ly::SLAB);
                    tma_load_3d(tiles + st * Ly::TILE, map, c * 64, unit.g, unit.first + j * BM, full);
                    last_bar = full, last_parity = (i / ST) & 1;
                }
            } else if (role < 4 && (role == 2 ? unit.last[0] : unit.last[1]) >= 0) {
                const int s = role - 2;
                const uint32_t use = s ? taken[1] : taken[0];
                ok = wait(q_empty(s, use), ((use / QB) & 1) ^ 1);
                if (ok) {
                    last_bar = q_full(s, use), last_parity = (use / QB) & 1;
                    mbar_expect_tx(last_bar, Ly::SLAB);
                    tma_load_3d(q_tile(s, use) + c * Ly::SLAB, &map_q, c * 64, s ? unit.head[1] : unit.head[0],
                                unit.first + (s ? unit.token[1] : unit.token[0]), last_bar);
                }
            }
            it += nb;
#pragma unroll
            for (int s = 0; s < 2; s++) taken[s] += unit.last[s] >= 0;
            if (!__all_sync(0xffffffffu, ok)) break;
            int got = 0;
            uint32_t x = 0;
            if (lane == 0) {
                ok = wait(next_full, n & 1);
                if (ok)
                    asm volatile(
                        "{\n\t.reg .pred q;\n\t.reg .b128 h;\n\t"
                        "ld.shared.b128 h, [%2];\n\t"
                        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 q, h;\n\t"
                        "selp.u32 %0, 1, 0, q;\n\t"
                        "mov.u32 %1, 0;\n\t"
                        "@q clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
                        : "=r"(got), "=r"(x)
                        : "r"(next_at)
                        : "memory");
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            if (!ok) break;
            got = __shfl_sync(0xffffffffu, got, 0);
            x = __shfl_sync(0xffffffffu, x, 0);
            more = got && list.find(p, x, unit);  // the end goes through the list as a unit without rows
        }
        if (!ok) give_up();
        // given up: let this lane's last copy, and an answer, land before the shared memory is another's
        if (*abort_flag && last_bar)
            for (uint32_t i = 0; i < 1000u && !mbar_try_wait(last_bar, last_parity); i++) {
            }
        if (*abort_flag && lane == 0)
            for (uint32_t i = 0; i < 10u && !mbar_try_wait(next_full, n & 1); i++) {
            }
    } else if (warp == 9) {
        // ---------------- products ----------------
        // One lane, chosen by elect.sync: the compiler then knows that the operands are the warp's only ones and takes
        // them into uniform registers.  (Under `lane == 0` each product took about 120 cycles to issue, twice what it
        // takes to execute.)
        if (elect_one()) {
            constexpr uint32_t id_s = idesc_f16(BF, BM, 0), id_o = idesc_f16(BF, HD, 1);
            // The units' blocks are one stream.  head_dim 64: block k + 1's scores go before block k's values, as soon as
            // softmax has read the scores of block k.  128: after them, side by side, since block k's p lies in their
            // place (products of one CTA execute in issue order).
            struct Block {
                int j, n0, n1;                  // block of its unit, and the unit's blocks on either side
                __device__ bool has(int s) const { return j < (s ? n1 : n0); }
                __device__ bool last(int s) const { return j + 1 == (s ? n1 : n0); }
            };
            uint32_t n = 0, k_it = 0, v_it = 0;               // units, blocks of K and of V taken
            uint32_t sc0 = 0, sc1 = 0, vc0 = 0, vc1 = 0;      // scores and values of either side so far
            uint32_t tq0 = 0, tq1 = 0, tv0 = 0, tv1 = 0;      // tiles of either side begun, for the scores and the values
            bool ok = true, more = true;
            Block next{-1, 0, 0}, now{0, 0, 0};
            // The stream's next block into `next`; false at its end.
            auto advance = [&]() {
                if (++next.j < max(next.n0, next.n1)) return true;
                const int slot = n % kSlots;
                ok = wait(u_full(slot), (n / kSlots) & 1);
                if (!ok) return false;
                n++;
                const int len = units[slot].len;
                next.j = 0, next.n0 = units[slot].last[0] + 1, next.n1 = units[slot].last[1] + 1;
                mbar_arrive(u_empty(slot));
                return len != 0;
            };
            // S_s = Q_s K^T of block `next`
            auto scores = [&](int s) {
                const uint32_t use = s ? tq1 : tq0, st = k_it % ST, done = s ? sc1 : sc0;
                if (next.j == 0) ok = ok && wait(q_full(s, use), (use / QB) & 1);
                if (Ly::OWN_P) ok = ok && wait(s_free(s), (done & 1) ^ 1);
                if (!ok) return;
                tc_fence_after();
                const uint64_t a = desc_sw128(q_tile(s, use), 0), b = desc_sw128(base + Ly::K_OFF + st * Ly::TILE, 0);
#pragma unroll
                for (int kk = 0; kk < HD / 16; kk++)
                    mma_ss(tmem + Ly::S + s * 128, a + (kk / 4) * (Ly::SLAB >> 4) + 2 * (kk % 4),
                           b + (kk / 4) * (Ly::SLAB >> 4) + 2 * (kk % 4), id_s, kk > 0);
                mma_commit(s_full(s));
                if (next.last(s)) {
                    mma_commit(q_empty(s, use));
                    s ? tq1++ : tq0++;
                }
                s ? sc1++ : sc0++;
            };
            // O_s += P_s V of block `now`, its keys in two halves
            auto values = [&](int s) {
                const uint32_t done = s ? vc1 : vc0, st = v_it % ST;
                if (now.j == 0) ok = ok && wait(o_free(s), ((s ? tv1 : tv0) & 1) ^ 1);
                const uint64_t b = desc_sw128(base + Ly::V_OFF + st * Ly::TILE, Ly::SLAB);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    ok = ok && wait(half ? p_full(s) : p_half(s), done & 1);
                    if (!ok) return;
                    tc_fence_after();
#pragma unroll
                    for (int kk = BM / 32 * half; kk < BM / 32 * (half + 1); kk++)
                        mma_ts(tmem + Ly::O + s * HD, tmem + Ly::P + s * Ly::P_STEP + 8 * kk, b + 128 * kk, id_o,
                               now.j > 0 || kk > 0);
                }
                mma_commit(o_full(s));
                if (now.last(s)) s ? tv1++ : tv0++;
                s ? vc1++ : vc0++;
            };
            for (bool begun = false; more || begun; begun = true) {
                // head_dim 64: scores of the next block of both sides, then values of this one; 128: side by side
                if (begun) now = next;
                more = more && advance();
                if (!ok) break;
                if (more) ok = wait(k_full(k_it % ST), (k_it / ST) & 1);
                if (more && Ly::OWN_P) {
#pragma unroll 1
                    for (int s = 0; s < 2; s++)
                        if (next.has(s)) scores(s);
                    mma_commit(k_empty(k_it % ST)), k_it++;
                }
                if (begun) ok = ok && wait(v_good(v_it % ST), (v_it / ST) & 1);
#pragma unroll 1
                for (int s = 0; s < 2; s++) {
                    if (begun && now.has(s)) values(s);
                    if (more && !Ly::OWN_P && next.has(s)) scores(s);
                }
                if (!ok) break;
                if (begun) mma_commit(v_empty(v_it % ST)), v_it++;
                if (!more) break;
                if (!Ly::OWN_P) mma_commit(k_empty(k_it % ST)), k_it++;
            }
            if (!ok) give_up();
        }
        __syncwarp();
    } else if (warp == 10) {
        // ---------------- V blocks on the diagonal ----------------
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t n = 0; ok; n++) {
            const int slot = n % kSlots;
            ok = __all_sync(0xffffffffu, wait(u_full(slot), (n / kSlots) & 1));
            if (!ok) break;
            Unit u;
            take(slot, u);
            if (u.len == 0) break;
            const int nb = u.blocks();
            bool bad = false;
#pragma unroll 1
            for (int j = 0; j < nb; j++) {
                const uint32_t i = it + j, st = i % ST;
                ok = __all_sync(0xffffffffu, wait(v_full(st), (i / ST) & 1));
                if (!ok) break;
                if (j == u.last[0] || j == u.last[1]) {
                    const int rows = min(BM, u.len - j * BM);
                    constexpr uint32_t EXP = BF ? 0x7f807f80u : 0x7c007c00u, ONE = BF ? 0x00800080u : 0x04000400u;
                    uint4* tile = reinterpret_cast<uint4*>(smem + Ly::V_OFF + st * Ly::TILE);
                    uint32_t seen = 0;
#pragma unroll 4
                    for (int x = lane; x < Ly::TILE / 16; x += 32) {
                        if ((x >> 3) % BM < rows) {  // 8 vectors a row, BM rows a slab
                            const uint4 w = tile[x];
                            // an all-ones exponent carries into the sign's place
                            seen |= ((w.x & EXP) + ONE) | ((w.y & EXP) + ONE) | ((w.z & EXP) + ONE) | ((w.w & EXP) + ONE);
                        } else {
                            tile[x] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    if (seen & 0x80008000u) {
                        auto finite = [&](uint32_t x) { return x & ~(((((x & EXP) + ONE) & 0x80008000u) >> 15) * 0xffffu); };
                        bad = true;
#pragma unroll 1
                        for (int x = lane; x < Ly::TILE / 16; x += 32)
                            tile[x] = make_uint4(finite(tile[x].x), finite(tile[x].y), finite(tile[x].z), finite(tile[x].w));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(v_good(st));
                    mbar_arrive(v_empty(st));
                }
            }
            if (!ok) break;
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) {
                if (bad) units[slot].bad = 1;
                mbar_arrive(u_seen(slot));
                mbar_arrive(u_empty(slot));
            }
            it += nb;
        }
        if (!ok) give_up();
    }
    } else {
        // ---------------- softmax, output ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int s = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + Ly::S + s * 128, tp = tmem + lanes + Ly::P + s * Ly::P_STEP,
                       to = tmem + lanes + Ly::O + s * HD;
        const float c = p.scale * 1.4426950408889634f;  // log2 e
        constexpr float RISE = BF ? 8.0f : 6.0f, LIFT = BF ? 0.0f : 15.0f - RISE;  // p = 2^(LIFT + x) with x <= RISE
        uint32_t cs = 0;  // blocks of this side
        float m = -INFINITY, off = 0.0f, l = 0.0f;  // maximum that exponents refer to, LIFT - c m, row sum
        auto wait_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        // A higher maximum: l and, where there is one, O scaled down to it.
        auto raise = [&](float to_m, bool scale_o) {
            const float f = to_m == m ? 1.0f : ex2((m - to_m) * c);
            m = to_m;
            off = m == -INFINITY ? 0.0f : BF ? -m * c : fmaf(-m, c, LIFT);
            l *= f;
            if (!scale_o) return;
#pragma unroll 1
            for (int q = 0; q < HD; q += 16) {
                uint32_t o[16];
                tmem_ld16(to + q, o);
                tmem_wait_ld();
#pragma unroll
                for (int w = 0; w < 16; w++) o[w] = __float_as_uint(__uint_as_float(o[w]) * f);
                tmem_st16(to + q, o);
            }
        };
        // This warp's p of half a block is in TMEM.
        auto publish = [&](uint32_t bar) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if(bar, lane == 0);
        };
        bool ok = true;
        for (uint32_t n = 0; ok; n++) {
            const int slot = n % kSlots;
            ok = wait_all(u_full(slot), (n / kSlots) & 1);
            if (!ok) break;
            const int first = units[slot].first, len = units[slot].len, token0 = units[slot].token[s],
                      head0 = units[slot].head[s], nb = units[slot].last[s] + 1;
            if (len == 0) break;
            m = -INFINITY, off = 0.0f, l = 0.0f;
#pragma unroll 1
            for (int j = 0; j < nb; j++) {
                ok = wait_all(s_full(s), (cs + j) & 1);
                if (!ok) break;
                tc_fence_after();
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                uint32_t r[128];
                // r holds the block's quarters in order; on the diagonal from the warp's own quarter on, so that the one to mask
                // by lane has fixed registers
                // (the warp's 32 rows end in one quarter, as 128 / F tokens and their starts are multiples of each other)
                const int end = (token0 & (BM - 1)) + ((threadIdx.x & 127) >> p.pack);  // last key that the row sees there
                const uint32_t turn = j == nb - 1 ? end >> 5 : 0;
#pragma unroll
                for (int q = 0; q < 4; q++) tmem_ld32(ts + 32 * ((turn + q) & 3), r + 32 * q);
                tmem_wait_ld();
                if (Ly::OWN_P) {
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_if(s_free(s), lane == 0);
                }
                const bool diagonal = j == nb - 1;
                if (diagonal) {  // r[0 .. 31] are the quarter where this warp's rows end; those behind it are not seen at all
#pragma unroll
                    for (int q = 0; q < 32; q++)
                        if (q > (end & 31)) r[q] = 0xff800000u;
#pragma unroll
                    for (int q = 32; q < 128; q++)
                        if ((end >> 5) + q / 32 < 4) r[q] = 0xff800000u;
                }
                const float top = row_max<128>(r);
                const bool rise = (top - m) * c > RISE;  // true of a first block that has a score
                const bool any_rise = __any_sync(0xffffffffu, rise);
                // P's columns (head_dim 64) and O are free once the product before is done
                if (j > 0 && (Ly::OWN_P || any_rise)) {
                    ok = wait_all(o_full(s), (cs + j - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                }
                if (any_rise) raise(rise ? top : m, j > 0);
                uint32_t pk[2][16];
                if (Ly::OWN_P && diagonal && end < 64) {  // nothing behind the block's first half is seen
                    exponentials<T>(r, c, off, sum, pk[0]);
                    tmem_st16(tp + 16 * turn, pk[0]);
#pragma unroll
                    for (int q = 0; q < 16; q++) pk[0][q] = pk[1][q] = 0;
                    tmem_st16(tp + 32, pk[0]);
                    tmem_st16(tp + 48, pk[0]);
                    if (turn) exponentials<T>(r + 96, c, off, sum, pk[1]);
                    tmem_st16(tp + 16 * (turn ^ 1), pk[1]);
                    publish(p_full(s));
                    mbar_arrive_if(p_half(s), lane == 0);
                } else {
                    exponentials<T>(r, c, off, sum, pk[0]);
                    tmem_st16(tp + 16 * turn, pk[0]);
                    exponentials<T>(r + 32, c, off, sum, pk[1]);
                    tmem_st16(tp + 16 * ((turn + 1) & 3), pk[1]);
                    exponentials<T>(r + 64, c, off, sum, pk[0]);
                    if (!diagonal) publish(p_half(s));  // its stores went on while this quarter was computed
                    tmem_st16(tp + 16 * ((turn + 2) & 3), pk[0]);
                    exponentials<T>(r + 96, c, off, sum, pk[1]);
                    tmem_st16(tp + 16 * ((turn + 3) & 3), pk[1]);
                    publish(p_full(s));
                    if (diagonal) mbar_arrive_if(p_half(s), lane == 0);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            ok = ok && wait_all(u_seen(slot), (n / kSlots) & 1);
            if (!ok) break;
            if (nb) {
                const int bad = units[slot].bad;
                ok = wait_all(o_full(s), (cs + nb - 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int row0 = (warp & 3) * 32;  // this warp's first row of the tile
                const int tokens = len - token0, heads = (1 << p.pack) - 1;
                T* out = static_cast<T*>(p.out) + ((int64_t)first + token0) * p.out_stride + head0 * HD;
                uint4* stage = reinterpret_cast<uint4*>(smem + Ly::OUT_OFF + warp * 4096);
#pragma unroll 1
                for (int q = 0; q < HD; q += 64) {
                    uint32_t o[64];
                    tmem_ld32(to + q, o);
                    tmem_ld32(to + q + 32, o + 32);
                    tmem_wait_ld();
                    if (q + 64 == HD) {
                        tc_fence_before();
                        __syncwarp();
                        mbar_arrive_if(o_free(s), lane == 0);
                    }
                    // a row's 128 bytes by its own thread, chunks permuted by the row against bank conflicts; then
                    // eight lanes store one row
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            y[e] = pack2<T>(__uint_as_float(o[8 * x + 2 * e]) * inv, __uint_as_float(o[8 * x + 2 * e + 1]) * inv);
                        stage[lane * 8 + (x ^ (lane & 7))] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int w = 0; w < 8; w++) {
                        const int r = 4 * w + (lane >> 3), token = (row0 + r) >> p.pack, head = (row0 + r) & heads;
                        if (token < tokens)
                            *reinterpret_cast<uint4*>(out + token * p.out_stride + head * HD + q + 8 * (lane & 7)) =
                                stage[r * 8 + ((lane & 7) ^ (r & 7))];
                    }
                    __syncwarp();
                }
                if (bad)
                    for (int w = row0; w < row0 + 32; w++) {
                        const int token = token0 + (w >> p.pack), head = head0 + (w & heads);
                        if (token < len) add_nonfinite<T, HD>(p, first, token, head, head / (p.packs << p.pack), token0);
                    }
            }
            __syncwarp();
            mbar_arrive_if(u_empty(slot), lane == 0);
            cs += nb;
        }
        if (!ok) give_up();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

pf_status get_encode(EncodeTiled* fn) {
    static std::mutex mu;
    static EncodeTiled cached = nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!cached) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        PF_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q));
        PF_CHECK(f && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled unavailable");
        cached = reinterpret_cast<EncodeTiled>(f);
    }
    *fn = cached;
    return PF_OK;
}

// Boxes of 64 columns x `heads` heads x 128 / heads tokens of 16-bit values; tokens past the end read as zeros.
pf_status make_map(CUtensorMap* map, const void* at, int hd, int64_t n_heads, int64_t tokens, int64_t stride, int heads) {
    EncodeTiled enc;
    PF_TRY(get_encode(&enc));
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)n_heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)(BM / heads)}, estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(at), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    PF_CHECK(r == CUDA_SUCCESS, "pf_prompt_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return PF_OK;
}

template <typename T, int HD>
pf_status launch_prompt(const PromptParams& p, cudaStream_t st) {
    using Ly = Layout<HD>;
    CUtensorMap mq, mk, mv;
    PF_TRY(make_map(&mq, p.q, HD, p.n_heads, p.n_tokens, p.q_stride, 1 << p.pack));
    PF_TRY(make_map(&mk, p.k, HD, p.n_kv_heads, p.n_tokens, p.k_stride, 1));
    PF_TRY(make_map(&mv, p.v, HD, p.n_kv_heads, p.n_tokens, p.v_stride, 1));
    // tiles: sum ceil(len / T) <= (sum len + (T - 1) n_seqs) / T, and half a pair more a sequence if a kv head's are odd
    const int64_t tokens = BM >> p.pack, tiles = ((int64_t)p.n_tokens + (tokens - 1) * p.n_seqs) / tokens;
    const int64_t units = p.n_kv_heads * ((tiles * p.packs + (p.packs % 2 ? p.n_seqs : 0)) / 2);
    PF_CHECK(units <= INT32_MAX, "pf_prompt_attention: too many row tiles");
    if (units == 0) return PF_OK;  // not one sequence can hold a row
    static std::atomic<uint64_t> attr{0};
    PF_TRY(raise_smem_limit(prompt_kernel<T, HD>, Ly::SMEM, attr));
    return launch_after("prompt_attention", prompt_kernel<T, HD>, dim3((unsigned)units), kThreads, Ly::SMEM, st, mq, mk, mv, p);
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
    PF_CHECK(n_seqs >= 0 && n_tokens >= 0 && n_seqs <= 1 << 20 && n_tokens <= 1 << 30,
             "pf_prompt_attention: %d sequences, %d tokens", n_seqs, n_tokens);
    PF_CHECK(n_kv_heads > 0 && n_heads > 0 && n_heads <= 65535 && n_heads % n_kv_heads == 0,
             "pf_prompt_attention: %d heads over %d kv heads", n_heads, n_kv_heads);
    PF_CHECK(scale > 0.0f && scale <= kMaxScale, "pf_prompt_attention: scale must be positive and at most 2.3e38");
    const int64_t wq = (int64_t)n_heads * head_dim, wk = (int64_t)n_kv_heads * head_dim;
    PF_CHECK(q_stride >= wq && out_stride >= wq && k_stride >= wk && v_stride >= wk,
             "pf_prompt_attention: a stride is smaller than its row");
    PF_CHECK(((q_stride | k_stride | v_stride | out_stride) % 8) == 0 &&
                 (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16) == 0,
             "pf_prompt_attention: pointers and strides must be multiples of 16 bytes");
    PF_CHECK(std::max(std::max(q_stride, out_stride), std::max(k_stride, v_stride)) < (int64_t)1 << 38,
             "pf_prompt_attention: a stride is too large");  // a tensor map's strides end at 2^40 bytes
    PF_CHECK((uintptr_t)offsets % 4 == 0, "pf_prompt_attention: offsets must be 4-byte aligned");
    PF_TRY(require_device());
    if (n_seqs == 0 || n_tokens == 0) return PF_OK;
    PF_CHECK(q && k && v && out && offsets, "pf_prompt_attention: null argument");
    const int group = n_heads / n_kv_heads;
    int pack = 0;
    while (pack < 5 && group % (2 << pack) == 0) pack++;
    const PromptParams p{q, k, v, out, q_stride, k_stride, v_stride, out_stride, offsets, n_seqs, n_tokens, n_heads,
                         n_kv_heads, pack, group >> pack, scale, device_error_flag()};
    cudaStream_t st = as_stream(stream);
    if (dtype == PF_BF16)
        return head_dim == 64 ? launch_prompt<__nv_bfloat16, 64>(p, st) : launch_prompt<__nv_bfloat16, 128>(p, st);
    return head_dim == 64 ? launch_prompt<__half, 64>(p, st) : launch_prompt<__half, 128>(p, st);
}
