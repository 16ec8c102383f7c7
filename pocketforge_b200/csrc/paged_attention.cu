// paged_attention.cu — attention of the newest tokens over the paged cache.
#include "paged.cuh"
#include "row_attention.cuh"

namespace pf {

namespace {

struct PagedParams {
    pf_paged_cache c;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int layer, n_seqs, rows, n_heads;
    float scale;
    uint32_t* err;
};

// One warp a (sequence, row, head).
template <typename QT, typename CT, int HD>
__global__ void __launch_bounds__(32) paged_rows_kernel(const PagedParams p) {
    constexpr int N = HD / 32;
    const pf_paged_cache& c = p.c;
    const int lane = threadIdx.x, h = blockIdx.y, g = h / (p.n_heads / c.n_kv_heads);
    const int64_t i = blockIdx.x;
    const int b = (int)(i / p.rows), r = (int)(i % p.rows);
    const int n = seq_len(c, b, p.err) - p.rows + 1 + r;
    float q[N];
#pragma unroll
    for (int d = 0; d < N; d++) q[d] = (float)static_cast<const QT*>(p.q)[i * p.q_stride + h * HD + lane + 32 * d] * p.scale;
    RowSoftmax<HD> s;
    for (int j = 0; j < n; j++) {
        const int page = c.table[(int64_t)b * c.max_pages + j / c.page_size];
        if ((unsigned)page >= (unsigned)c.n_pages) {
            latch(p.err, ERR_BOUNDS);
            continue;
        }
        const int64_t row = slot_row(c, page, p.layer, g, j % c.page_size);
        const float ks = sizeof(CT) == 1 ? c.k_scale[row] : 1.0f, vs = sizeof(CT) == 1 ? c.v_scale[row] : 1.0f;
        float k[N], v[N];
#pragma unroll
        for (int d = 0; d < N; d++) {
            k[d] = (float)static_cast<const CT*>(c.k)[row * HD + lane + 32 * d] * ks;
            v[d] = (float)static_cast<const CT*>(c.v)[row * HD + lane + 32 * d] * vs;
        }
        s.add(warp_dot(q, k), v);
    }
#pragma unroll
    for (int d = 0; d < N; d++)
        static_cast<QT*>(p.out)[i * p.out_stride + h * HD + lane + 32 * d] = (QT)(s.l == 0.0f ? 0.0f : s.o[d] / s.l);
}

template <typename QT, typename CT>
pf_status launch_paged(const PagedParams& p, cudaStream_t st) {
    const dim3 grid(p.n_seqs * p.rows, p.n_heads);
    if (p.c.head_dim == 64) paged_rows_kernel<QT, CT, 64><<<grid, 32, 0, st>>>(p);
    else paged_rows_kernel<QT, CT, 128><<<grid, 32, 0, st>>>(p);
    return launch_check("paged_attention");
}

}  // namespace

}  // namespace pf

using namespace pf;

extern "C" {

size_t pf_paged_attention_work_bytes(const pf_paged_cache* c, int32_t n_seqs, int32_t rows, int32_t n_heads) {
    if (!c || n_seqs < 0 || rows < 1 || rows > 8 || n_heads < 1 || c->n_kv_heads < 1 || n_heads % c->n_kv_heads) return 0;
    return 16;
}

pf_status pf_paged_attention(const pf_paged_cache* c, int32_t layer, const void* q, int64_t q_stride, void* out,
                             int64_t out_stride, int32_t dtype, int32_t n_seqs, int32_t rows, int32_t n_heads,
                             float scale, void* work, size_t work_bytes, void* stream) {
    PF_TRY(check_paged_cache(c, "pf_paged_attention", false));
    PF_CHECK(layer >= 0 && layer < c->n_layers, "pf_paged_attention: layer %d of %d", layer, c->n_layers);
    PF_CHECK(n_seqs >= 0 && n_seqs <= c->max_seqs, "pf_paged_attention: %d sequences of %d", n_seqs, c->max_seqs);
    PF_CHECK(rows >= 1 && rows <= 8, "pf_paged_attention: %d rows are not 1 to 8", rows);
    PF_CHECK(n_heads > 0 && n_heads <= 65535 && n_heads % c->n_kv_heads == 0,
             "pf_paged_attention: %d heads over %d kv heads", n_heads, c->n_kv_heads);
    PF_CHECK(c->dtype == PF_I8 ? dtype == PF_F32 || dtype == PF_BF16 || dtype == PF_F16 : dtype == c->dtype,
             "pf_paged_attention: rows of dtype %d over a cache of dtype %d", dtype, c->dtype);
    PF_CHECK(scale > 0.0f && scale <= 3.402823466e38f, "pf_paged_attention: scale must be positive and finite");
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
    PagedParams p{*c, q, out, q_stride, out_stride, layer, n_seqs, rows, n_heads, scale, device_error_flag()};
    cudaStream_t st = as_stream(stream);
    if (c->dtype == PF_BF16) return launch_paged<__nv_bfloat16, __nv_bfloat16>(p, st);
    if (c->dtype == PF_F16) return launch_paged<__half, __half>(p, st);
    if (dtype == PF_F32) return launch_paged<float, int8_t>(p, st);
    if (dtype == PF_BF16) return launch_paged<__nv_bfloat16, int8_t>(p, st);
    return launch_paged<__half, int8_t>(p, st);
}

}  // extern "C"
