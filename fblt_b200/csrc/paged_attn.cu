// Attention of new query rows over the 8-bit paged KV cache (fblt_paged_attn).
#include "paged.cuh"

namespace fblt {

struct PagedAttnParams {
    PagedView pv;
    int batch, H, G, total, max_new, block_mode, window;
    const int32_t *cu, *base;
    const float *q;
    int64_t qs;
    float *out;
    int64_t os;
    float qscale; // scale * log2(e)
};

// One warp per (row, query head): keys one after the other, lanes over head_dim.
template <int HD, int FMT>
__global__ void __launch_bounds__(128) paged_row_kernel(const PagedAttnParams p) {
    constexpr int E = HD / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x * 4 + warp;
    int r0, n, base;
    if (!paged_seq(p.pv, p.cu, p.base, p.total, b, r0, n, base)) return;
    if (n > p.max_new && i == 0 && h == 0 && lane == 0) p.pv.raise(FBLT_PAGED_BAD_LENGTH);
    if (i >= n) return;
    const int pos = base + i, kvh = h / p.G;
    const int hi = p.block_mode ? base + n : pos + 1;
    const int lo = !p.block_mode && p.window > 0 ? max(0, pos - p.window + 1) : 0;
    float q[E], acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = p.q[(int64_t)(r0 + i) * p.qs + h * HD + lane * E + e] * p.qscale;
        acc[e] = 0.0f;
    }
    for (int j = lo; j < hi; ++j) {
        const int pi = j / p.pv.page_size, page = p.pv.page(b, pi);
        if (page < 0) {
            if (lane == 0) p.pv.raise(FBLT_PAGED_BAD_PAGE);
            continue;
        }
        const int64_t at = p.pv.row(page, kvh, j - pi * p.pv.page_size);
        const float ks = kv_scale<FMT>(p.pv.ke[at]), vs = kv_scale<FMT>(p.pv.ve[at]);
        float s = 0.0f, v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t c = at * HD + lane * E + e;
            s += q[e] * (kv_values<FMT>(p.pv.kc[c], 1.0f).x * ks);
            v[e] = kv_values<FMT>(p.pv.vc[c], 1.0f).x * vs;
        }
        s = warp_sum(s);
        if (!finite_f(s)) continue;
        const float mn = fmaxf(m, s), c = exp2f(m - mn), w = exp2f(s - mn);
        m = mn;
        l = l * c + w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + w * v[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) p.out[(int64_t)(r0 + i) * p.os + h * HD + lane * E + e] = l > 0.0f ? acc[e] / l : 0.0f;
}

int paged_attn_check(const fblt_paged_attn_desc *d) {
    const char *who = "paged_attn";
    if (!d) return fail(FBLT_ERR_ARG, "%s: NULL descriptor", who);
    if (d->batch < 0 || d->total_rows < 0 || d->max_new < 0 || d->max_len < 0) return fail(FBLT_ERR_ARG, "%s: negative size", who);
    int st = validate_paged_cache(d->cache, d->batch, who);
    if (st != FBLT_OK) return st;
    if (d->num_heads < 1 || d->num_heads > 65535 || d->num_heads % d->cache.num_kv_heads)
        return fail(FBLT_ERR_ARG, "%s: num_heads %d is not a multiple of num_kv_heads %d (at most 65535)", who, d->num_heads,
                    d->cache.num_kv_heads);
    if (d->window < 0) return fail(FBLT_ERR_ARG, "%s: negative window", who);
    if (d->splits < 0) return fail(FBLT_ERR_ARG, "%s: negative splits", who);
    if (!(fabsf(d->scale) < INFINITY)) return fail(FBLT_ERR_ARG, "%s: scale must be finite", who);
    if (d->batch > 65535) return fail(FBLT_ERR_LIMIT, "%s: batch exceeds 65535 per launch", who);
    if (d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return FBLT_OK;
    if (!d->cu_new || !d->base_len || !d->q || !d->out) return fail(FBLT_ERR_ARG, "%s: NULL buffer", who);
    const int64_t E = (int64_t)d->num_heads * d->cache.head_dim;
    if (d->q_stride < E || d->out_stride < E) return fail(FBLT_ERR_ARG, "%s: row stride smaller than num_heads*head_dim", who);
    if ((d->q_stride | d->out_stride) & 3) return fail(FBLT_ERR_ARG, "%s: strides must be multiples of 4 elements", who);
    if (((uintptr_t)d->q | (uintptr_t)d->out) & 15) return fail(FBLT_ERR_ARG, "%s: buffers must be 16-byte aligned", who);
    return FBLT_OK;
}

template <int HD, int FMT>
static int launch_paged_row(const PagedAttnParams &p, cudaStream_t s) {
    const dim3 grid((unsigned)((p.max_new + 3) / 4), (unsigned)p.H, (unsigned)p.batch);
    paged_row_kernel<HD, FMT><<<grid, 128, 0, s>>>(p);
    count_launch();
    return check_launch("paged_row_kernel");
}

} // namespace fblt

extern "C" size_t fblt_paged_attn_workspace(const fblt_paged_attn_desc *d) {
    if (fblt::paged_attn_check(d) != FBLT_OK) return 0;
    return 0;
}

extern "C" int fblt_paged_attn(const fblt_paged_attn_desc *d, void *workspace, size_t workspace_bytes, void *stream) {
    fblt::NvtxRange nvtx_range("fblt_paged_attn");
    using namespace fblt;
    (void)workspace;
    (void)workspace_bytes;
    int st = paged_attn_check(d);
    if (st != FBLT_OK) return st;
    if (d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return FBLT_OK;
    PagedAttnParams p;
    memset(&p, 0, sizeof(p));
    p.pv = paged_view(d->cache);
    p.batch = d->batch;
    p.H = d->num_heads;
    p.G = d->num_heads / d->cache.num_kv_heads;
    p.total = d->total_rows;
    p.max_new = d->max_new;
    p.block_mode = d->block_mode ? 1 : 0;
    p.window = d->window;
    p.cu = d->cu_new;
    p.base = d->base_len;
    p.q = d->q;
    p.qs = d->q_stride;
    p.out = d->out;
    p.os = d->out_stride;
    p.qscale = d->scale * kLog2e;
    cudaStream_t s = (cudaStream_t)stream;
    const bool e4 = d->cache.format == FBLT_KV_E4M3;
    switch (d->cache.head_dim) {
    case 32: return e4 ? launch_paged_row<32, FBLT_KV_E4M3>(p, s) : launch_paged_row<32, FBLT_KV_INT8>(p, s);
    case 64: return e4 ? launch_paged_row<64, FBLT_KV_E4M3>(p, s) : launch_paged_row<64, FBLT_KV_INT8>(p, s);
    default: return e4 ? launch_paged_row<128, FBLT_KV_E4M3>(p, s) : launch_paged_row<128, FBLT_KV_INT8>(p, s);
    }
}
