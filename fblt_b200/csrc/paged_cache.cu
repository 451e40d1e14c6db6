// Rows in and out of the 8-bit paged KV cache: per-head norm + rotation (fblt_qk_norm_rope), the same with K and V
// quantised into their pages (fblt_paged_append), and the way back (fblt_paged_read).
//
// All three are one pass over the data: head_dim / 4 lanes hold one (row, head) in registers, four values each, so the
// sum of squares and the largest magnitude are shuffles inside those lanes and nothing is read twice. What bounds
// them is HBM (reading and writing every value once).
#include "paged.cuh"

namespace fblt {

constexpr int kRowThreads = 256;
constexpr int kMaxRows = 16; // rows of one CTA

struct RowInfo {
    int pos;  // < 0: the row is not to be touched
    int page; // < 0: no page
    int slot;
    int b;
};

struct NormRopeParams {
    PagedView pv;     // append
    int64_t rows;
    int batch, qh, kh, rows_per_cta, rope_len;
    const float *q, *k, *v;
    int64_t qs, ks, vs;
    float *qo, *ko;
    int64_t qos, kos;
    const float *qg, *kg, *cs, *sn;
    float eps;
    const int32_t *pos;          // norm + rotation alone
    const int32_t *cu, *base;    // append
};

// Sequence, position and page of a packed row: the last b with cu[b] <= r.
__device__ __forceinline__ RowInfo find_row(const PagedView &pv, const int32_t *cu, const int32_t *base, int batch, int total,
                                            int r) {
    RowInfo ri;
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= r) lo = mid;
        else hi = mid;
    }
    ri.b = lo;
    ri.pos = ri.page = -1;
    ri.slot = 0;
    int r0, n, p0;
    if (!paged_seq(pv, cu, base, total, lo, r0, n, p0)) return ri;
    if (r < r0 || r >= r0 + n) {
        pv.raise(FBLT_PAGED_BAD_LENGTH);
        return ri;
    }
    ri.pos = p0 + (r - r0);
    const int pi = ri.pos / pv.page_size;
    ri.slot = ri.pos - pi * pv.page_size;
    ri.page = pv.page(lo, pi);
    if (ri.page < 0) pv.raise(FBLT_PAGED_BAD_PAGE);
    return ri;
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// FMT < 0: norm + rotation only. Otherwise units qh .. qh + kh are K, the next kh V, both quantised into the pages.
template <int HD, int FMT>
__global__ void __launch_bounds__(kRowThreads) norm_rope_kernel(const NormRopeParams p) {
    constexpr int LPH = HD / 4, GROUPS = kRowThreads / LPH, U = 2;
    constexpr bool APPEND = FMT >= 0;
    using F = KvFormat<(FMT >= 0 ? FMT : 0)>;
    __shared__ RowInfo info[kMaxRows];
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows_per_cta;
    const int nrows = (int)min((int64_t)p.rows_per_cta, p.rows - row0);
    if (tid < nrows) {
        if (APPEND) {
            info[tid] = find_row(p.pv, p.cu, p.base, p.batch, (int)p.rows, (int)row0 + tid);
        } else {
            RowInfo ri;
            ri.pos = p.pos ? p.pos[row0 + tid] : 0;
            ri.page = ri.slot = ri.b = 0;
            info[tid] = ri;
        }
        if (p.cs && (info[tid].pos < 0 ? !APPEND : info[tid].pos >= p.rope_len)) p.pv.raise(FBLT_PAGED_BAD_POSITION);
    }
    __syncthreads();
    const int units = p.qh + (APPEND ? 2 : 1) * p.kh, items = nrows * units;
    const int group = tid / LPH, lane = tid % LPH;
    for (int it0 = 0; it0 < items; it0 += GROUPS * U) { // the same trip count for every lane of a warp
        float4 x[U];
        int row[U], unit[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * GROUPS + group;
            row[u] = it < items ? it / units : 0;
            unit[u] = it < items ? it - row[u] * units : -1;
            if (APPEND && info[row[u]].pos < 0) unit[u] = -1;
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (unit[u] >= 0) {
                const int64_t r = row0 + row[u];
                const float *src = unit[u] < p.qh                  ? p.q + r * p.qs + (int64_t)unit[u] * HD
                                   : !APPEND || unit[u] < p.qh + p.kh ? p.k + r * p.ks + (int64_t)(unit[u] - p.qh) * HD
                                                                   : p.v + r * p.vs + (int64_t)(unit[u] - p.qh - p.kh) * HD;
                x[u] = *reinterpret_cast<const float4 *>(src + lane * 4);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool is_q = unit[u] < p.qh, is_v = APPEND && unit[u] >= p.qh + p.kh;
            const float *gain = is_v ? nullptr : is_q ? p.qg : p.kg;
            const float ss = group_sum<LPH>(x[u].x * x[u].x + x[u].y * x[u].y + (x[u].z * x[u].z + x[u].w * x[u].w));
            if (gain) {
                const float inv = __frsqrt_rn(ss * (1.0f / HD) + p.eps);
                const float4 g = __ldg(reinterpret_cast<const float4 *>(gain) + lane);
                x[u].x *= inv * g.x;
                x[u].y *= inv * g.y;
                x[u].z *= inv * g.z;
                x[u].w *= inv * g.w;
            }
            const int pos = info[row[u]].pos;
            if (p.cs && !is_v && unit[u] >= 0 && pos >= 0 && pos < p.rope_len)
                x[u] = rope_rotate4(x[u], p.cs, p.sn, pos, HD / 2, lane * 2);
            if (!APPEND || is_q) {
                if (unit[u] >= 0) {
                    const int64_t r = row0 + row[u];
                    float *dst = is_q ? p.qo + r * p.qos + (int64_t)unit[u] * HD : p.ko + r * p.kos + (int64_t)(unit[u] - p.qh) * HD;
                    *reinterpret_cast<float4 *>(dst + lane * 4) = x[u];
                }
            }
            if (APPEND) {
                // 0 for what is not finite: the exponent comes from the finite values
                const float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                float a = 0.0f;
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (finite_f(v[i])) a = fmaxf(a, fabsf(v[i]));
                    else odd = true;
                }
                const int e = F::exponent(group_max<LPH>(a));
                if (unit[u] >= 0 && !is_q) {
                    if (odd) p.pv.raise(FBLT_PAGED_NONFINITE);
                    const RowInfo ri = info[row[u]];
                    if (ri.page >= 0) {
                        const float s = exp2_int(-e), top = (float)F::kQmax;
                        float y[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = isnan(v[i]) ? 0.0f : fminf(fmaxf(v[i] * s, -top), top);
                        const int64_t at = p.pv.row(ri.page, unit[u] - p.qh - (is_v ? p.kh : 0), ri.slot);
                        uint8_t *code = (is_v ? p.pv.vc : p.pv.kc) + at * HD + lane * 4;
                        *reinterpret_cast<uint32_t *>(code) = F::codes(y[0], y[1], y[2], y[3]);
                        if (lane == 0) (is_v ? p.pv.ve : p.pv.ke)[at] = (int8_t)e;
                    }
                }
            }
        }
    }
}

struct ReadParams {
    PagedView pv;
    int rows, batch, rows_per_cta;
    const int32_t *cu, *start;
    void *ko, *vo;
    int64_t kos, vos;
};

template <int HD, int FMT, bool BF16>
__global__ void __launch_bounds__(kRowThreads) paged_read_kernel(const ReadParams p) {
    constexpr int LPH = HD / 4, GROUPS = kRowThreads / LPH, U = 4;
    __shared__ RowInfo info[kMaxRows];
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows_per_cta;
    const int nrows = (int)min((int64_t)p.rows_per_cta, p.rows - row0);
    if (tid < nrows) info[tid] = find_row(p.pv, p.cu, p.start, p.batch, p.rows, (int)row0 + tid);
    __syncthreads();
    const int kh = p.pv.kvh, skip = p.ko ? 0 : kh, units = (p.ko && p.vo ? 2 : 1) * kh, items = nrows * units;
    const int group = tid / LPH, lane = tid % LPH;
    for (int it0 = group; it0 < items; it0 += GROUPS * U) {
        uint32_t w[U];
        int row[U], unit[U], e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = it0 + u * GROUPS;
            row[u] = it < items ? it / units : 0;
            unit[u] = it < items ? it - row[u] * units + skip : -1;
            const RowInfo ri = info[row[u]];
            if (ri.pos < 0) unit[u] = -1;
            w[u] = 0;
            e[u] = 0;
            if (unit[u] >= 0 && ri.page >= 0) {
                const bool is_v = unit[u] >= kh;
                const int64_t at = p.pv.row(ri.page, unit[u] - (is_v ? kh : 0), ri.slot);
                w[u] = *reinterpret_cast<const uint32_t *>((is_v ? p.pv.vc : p.pv.kc) + at * HD + lane * 4);
                e[u] = (is_v ? p.pv.ve : p.pv.ke)[at];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (unit[u] < 0) continue;
            const bool is_v = unit[u] >= kh;
            const int64_t at = (row0 + row[u]) * (is_v ? p.vos : p.kos) + (int64_t)(unit[u] - (is_v ? kh : 0)) * HD + lane * 4;
            const float4 x = kv_values<FMT>(w[u], kv_scale<FMT>(e[u]));
            void *dst = is_v ? p.vo : p.ko;
            if (BF16) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
                uint2 o;
                o.x = *reinterpret_cast<const uint32_t *>(&lo);
                o.y = *reinterpret_cast<const uint32_t *>(&hi);
                *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(dst) + at) = o;
            } else {
                *reinterpret_cast<float4 *>(static_cast<float *>(dst) + at) = x;
            }
        }
    }
}

// Rows of one CTA: one while that fills the GPU, more when the launch is long anyway (the row look-up is then shared
// and the loop has loads to overlap).
static int rows_per_cta(int64_t rows) {
    const int64_t r = rows / (148 * 16);
    return r < 1 ? 1 : r > 8 ? 8 : (int)r;
}

static bool aligned16(const void *p) { return !(((uintptr_t)p) & 15); }

static int check_rows(const char *who, const char *what, const void *p, int64_t stride, int64_t cols) {
    if (!aligned16(p)) return fail(FBLT_ERR_ARG, "%s: %s must be 16-byte aligned", who, what);
    if (stride < cols) return fail(FBLT_ERR_ARG, "%s: %s row stride smaller than its heads * head_dim", who, what);
    if (stride & 3) return fail(FBLT_ERR_ARG, "%s: %s row stride must be a multiple of 4 elements", who, what);
    return FBLT_OK;
}

static int check_rope(const char *who, const float *cs, const float *sn, int rope_len) {
    if ((cs == nullptr) != (sn == nullptr)) return fail(FBLT_ERR_ARG, "%s: rope_cos and rope_sin go together", who);
    if (((uintptr_t)cs | (uintptr_t)sn) & 7) return fail(FBLT_ERR_ARG, "%s: rotary tables must be 8-byte aligned", who);
    if (cs && rope_len < 1) return fail(FBLT_ERR_ARG, "%s: rope_len must be given with the rotary tables", who);
    return FBLT_OK;
}

static int check_hd(const char *who, int hd) {
    if (hd != 32 && hd != 64 && hd != 128) return fail(FBLT_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64 or 128)", who, hd);
    return FBLT_OK;
}

int validate_paged_cache(const fblt_paged_cache &c, int batch, const char *who) {
    if (c.format != FBLT_KV_E4M3 && c.format != FBLT_KV_INT8) return fail(FBLT_ERR_ARG, "%s: unknown cache format %d", who, c.format);
    int st = check_hd(who, c.head_dim);
    if (st != FBLT_OK) return st;
    if (c.num_kv_heads < 1 || c.num_kv_heads > 1024) return fail(FBLT_ERR_ARG, "%s: num_kv_heads %d (1 .. 1024)", who, c.num_kv_heads);
    if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & 15))
        return fail(FBLT_ERR_UNSUPPORTED, "%s: page_size %d (a multiple of 16, 16 .. 1024)", who, c.page_size);
    if (c.num_pages < 0 || c.max_pages < 0) return fail(FBLT_ERR_ARG, "%s: negative page count", who);
    if (batch > 0) {
        if (!c.k_codes || !c.v_codes || !c.k_exp || !c.v_exp || !c.page_table) return fail(FBLT_ERR_ARG, "%s: NULL cache buffer", who);
        if (!aligned16(c.k_codes) || !aligned16(c.v_codes) || !aligned16(c.k_exp) || !aligned16(c.v_exp))
            return fail(FBLT_ERR_ARG, "%s: cache buffers must be 16-byte aligned", who);
        if (((uintptr_t)c.page_table | (uintptr_t)c.status) & 3) return fail(FBLT_ERR_ARG, "%s: page_table / status misaligned", who);
        if (c.page_table_stride < c.max_pages) return fail(FBLT_ERR_ARG, "%s: page_table_stride smaller than max_pages", who);
    }
    return FBLT_OK;
}

template <int HD, int FMT>
static int launch_norm_rope(NormRopeParams &p, cudaStream_t s, const char *what) {
    p.rows_per_cta = rows_per_cta(p.rows);
    const int64_t grid = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
    if (grid > INT_MAX) return fail(FBLT_ERR_LIMIT, "%s: too many rows", what);
    norm_rope_kernel<HD, FMT><<<(unsigned)grid, kRowThreads, 0, s>>>(p);
    count_launch();
    return check_launch(what);
}

template <int HD, int FMT>
static int launch_read(ReadParams &p, bool bf16, cudaStream_t s) {
    p.rows_per_cta = rows_per_cta(p.rows);
    const unsigned grid = (unsigned)((p.rows + p.rows_per_cta - 1) / p.rows_per_cta);
    if (bf16) paged_read_kernel<HD, FMT, true><<<grid, kRowThreads, 0, s>>>(p);
    else paged_read_kernel<HD, FMT, false><<<grid, kRowThreads, 0, s>>>(p);
    count_launch();
    return check_launch("paged_read_kernel");
}

int paged_append_check(const fblt_paged_append_desc *d) {
    const char *who = "paged_append";
    if (!d) return fail(FBLT_ERR_ARG, "%s: NULL descriptor", who);
    if (d->batch < 0 || d->total_rows < 0) return fail(FBLT_ERR_ARG, "%s: bad batch / total_rows", who);
    int st = validate_paged_cache(d->cache, d->batch, who);
    if (st != FBLT_OK) return st;
    if ((d->q == nullptr) != (d->q_out == nullptr)) return fail(FBLT_ERR_ARG, "%s: q and q_out go together", who);
    if (d->q && (d->num_heads < 1 || d->num_heads > 65536)) return fail(FBLT_ERR_ARG, "%s: bad num_heads", who);
    if (!aligned16(d->q_gain) || !aligned16(d->k_gain)) return fail(FBLT_ERR_ARG, "%s: gains must be 16-byte aligned", who);
    if ((d->q_gain || d->k_gain) && !(d->eps >= 0.0f && d->eps < INFINITY)) return fail(FBLT_ERR_ARG, "%s: eps must be finite and >= 0", who);
    if ((st = check_rope(who, d->rope_cos, d->rope_sin, d->rope_len)) != FBLT_OK) return st;
    if (d->batch == 0 || d->total_rows == 0) return FBLT_OK;
    if (!d->cu_new || !d->base_len || !d->k || !d->v) return fail(FBLT_ERR_ARG, "%s: NULL buffer", who);
    const int64_t qc = (int64_t)d->num_heads * d->cache.head_dim, kc = (int64_t)d->cache.num_kv_heads * d->cache.head_dim;
    if ((st = check_rows(who, "k", d->k, d->k_stride, kc)) != FBLT_OK) return st;
    if ((st = check_rows(who, "v", d->v, d->v_stride, kc)) != FBLT_OK) return st;
    if (d->q) {
        if ((st = check_rows(who, "q", d->q, d->q_stride, qc)) != FBLT_OK) return st;
        if ((st = check_rows(who, "q_out", d->q_out, d->q_out_stride, qc)) != FBLT_OK) return st;
        if (d->q == d->q_out && d->q_stride != d->q_out_stride) return fail(FBLT_ERR_ARG, "%s: in place needs one row stride", who);
    }
    return FBLT_OK;
}

} // namespace fblt

extern "C" int fblt_qk_norm_rope(const fblt_qk_norm_rope_desc *d, void *stream) {
    fblt::NvtxRange nvtx_range("fblt_qk_norm_rope");
    using namespace fblt;
    const char *who = "qk_norm_rope";
    if (!d) return fail(FBLT_ERR_ARG, "%s: NULL descriptor", who);
    int st = check_hd(who, d->head_dim);
    if (st != FBLT_OK) return st;
    if (d->rows < 0) return fail(FBLT_ERR_ARG, "%s: negative row count", who);
    if ((d->q == nullptr) != (d->q_out == nullptr) || (d->k == nullptr) != (d->k_out == nullptr))
        return fail(FBLT_ERR_ARG, "%s: q / q_out and k / k_out go together", who);
    if (!d->q && !d->k) return fail(FBLT_ERR_ARG, "%s: neither q nor k", who);
    if ((d->q && (d->num_heads < 1 || d->num_heads > 65536)) || (d->k && (d->num_kv_heads < 1 || d->num_kv_heads > 65536)))
        return fail(FBLT_ERR_ARG, "%s: bad head counts", who);
    const int64_t qc = (int64_t)d->num_heads * d->head_dim, kc = (int64_t)d->num_kv_heads * d->head_dim;
    if (d->q) {
        if ((st = check_rows(who, "q", d->q, d->q_stride, qc)) != FBLT_OK) return st;
        if ((st = check_rows(who, "q_out", d->q_out, d->q_out_stride, qc)) != FBLT_OK) return st;
        if (d->q == d->q_out && d->q_stride != d->q_out_stride) return fail(FBLT_ERR_ARG, "%s: in place needs one row stride", who);
    }
    if (d->k) {
        if ((st = check_rows(who, "k", d->k, d->k_stride, kc)) != FBLT_OK) return st;
        if ((st = check_rows(who, "k_out", d->k_out, d->k_out_stride, kc)) != FBLT_OK) return st;
        if (d->k == d->k_out && d->k_stride != d->k_out_stride) return fail(FBLT_ERR_ARG, "%s: in place needs one row stride", who);
    }
    if (!aligned16(d->q_gain) || !aligned16(d->k_gain)) return fail(FBLT_ERR_ARG, "%s: gains must be 16-byte aligned", who);
    if ((d->q_gain || d->k_gain) && !(d->eps >= 0.0f && d->eps < INFINITY)) return fail(FBLT_ERR_ARG, "%s: eps must be finite and >= 0", who);
    if ((st = check_rope(who, d->rope_cos, d->rope_sin, d->rope_len)) != FBLT_OK) return st;
    if (d->rope_cos && !d->pos) return fail(FBLT_ERR_ARG, "%s: rotary tables need positions", who);
    if (d->rows == 0) return FBLT_OK;
    NormRopeParams p;
    memset(&p, 0, sizeof(p));
    p.pv.status = d->status;
    p.rows = d->rows;
    p.qh = d->q ? d->num_heads : 0;
    p.kh = d->k ? d->num_kv_heads : 0;
    p.rope_len = d->rope_len;
    p.q = d->q;
    p.k = d->k;
    p.qs = d->q_stride;
    p.ks = d->k_stride;
    p.qo = d->q_out;
    p.ko = d->k_out;
    p.qos = d->q_out_stride;
    p.kos = d->k_out_stride;
    p.qg = d->q_gain;
    p.kg = d->k_gain;
    p.cs = d->rope_cos;
    p.sn = d->rope_sin;
    p.eps = d->eps;
    p.pos = d->rope_cos ? d->pos : nullptr;
    cudaStream_t s = (cudaStream_t)stream;
    switch (d->head_dim) {
    case 32: return launch_norm_rope<32, -1>(p, s, "norm_rope_kernel");
    case 64: return launch_norm_rope<64, -1>(p, s, "norm_rope_kernel");
    default: return launch_norm_rope<128, -1>(p, s, "norm_rope_kernel");
    }
}

extern "C" int fblt_paged_append(const fblt_paged_append_desc *d, void *stream) {
    fblt::NvtxRange nvtx_range("fblt_paged_append");
    using namespace fblt;
    const int st = paged_append_check(d);
    if (st != FBLT_OK) return st;
    if (d->batch == 0 || d->total_rows == 0) return FBLT_OK;
    NormRopeParams p;
    memset(&p, 0, sizeof(p));
    p.pv = paged_view(d->cache);
    p.rows = d->total_rows;
    p.batch = d->batch;
    p.qh = d->q ? d->num_heads : 0;
    p.kh = d->cache.num_kv_heads;
    p.rope_len = d->rope_len;
    p.q = d->q;
    p.k = d->k;
    p.v = d->v;
    p.qs = d->q_stride;
    p.ks = d->k_stride;
    p.vs = d->v_stride;
    p.qo = d->q_out;
    p.qos = d->q_out_stride;
    p.qg = d->q_gain;
    p.kg = d->k_gain;
    p.cs = d->rope_cos;
    p.sn = d->rope_sin;
    p.eps = d->eps;
    p.cu = d->cu_new;
    p.base = d->base_len;
    cudaStream_t s = (cudaStream_t)stream;
    const bool e4 = d->cache.format == FBLT_KV_E4M3;
    switch (d->cache.head_dim) {
    case 32: return e4 ? launch_norm_rope<32, FBLT_KV_E4M3>(p, s, "norm_rope_kernel") : launch_norm_rope<32, FBLT_KV_INT8>(p, s, "norm_rope_kernel");
    case 64: return e4 ? launch_norm_rope<64, FBLT_KV_E4M3>(p, s, "norm_rope_kernel") : launch_norm_rope<64, FBLT_KV_INT8>(p, s, "norm_rope_kernel");
    default: return e4 ? launch_norm_rope<128, FBLT_KV_E4M3>(p, s, "norm_rope_kernel") : launch_norm_rope<128, FBLT_KV_INT8>(p, s, "norm_rope_kernel");
    }
}

extern "C" int fblt_paged_read(const fblt_paged_read_desc *d, void *stream) {
    fblt::NvtxRange nvtx_range("fblt_paged_read");
    using namespace fblt;
    const char *who = "paged_read";
    if (!d) return fail(FBLT_ERR_ARG, "%s: NULL descriptor", who);
    if (d->batch < 0 || d->total_rows < 0) return fail(FBLT_ERR_ARG, "%s: bad batch / total_rows", who);
    int st = validate_paged_cache(d->cache, d->batch, who);
    if (st != FBLT_OK) return st;
    if (d->out_type != FBLT_PAGED_OUT_FP32 && d->out_type != FBLT_PAGED_OUT_BF16) return fail(FBLT_ERR_ARG, "%s: unknown out_type %d", who, d->out_type);
    if (!d->k_out && !d->v_out) return fail(FBLT_ERR_ARG, "%s: neither k_out nor v_out", who);
    if (d->batch == 0 || d->total_rows == 0) return FBLT_OK;
    if (!d->cu_rows) return fail(FBLT_ERR_ARG, "%s: NULL cu_rows", who);
    const bool bf16 = d->out_type == FBLT_PAGED_OUT_BF16;
    const int64_t kc = (int64_t)d->cache.num_kv_heads * d->cache.head_dim;
    if (d->k_out && (st = check_rows(who, "k_out", d->k_out, d->k_out_stride, kc)) != FBLT_OK) return st;
    if (d->v_out && (st = check_rows(who, "v_out", d->v_out, d->v_out_stride, kc)) != FBLT_OK) return st;
    if (bf16 && (((d->k_out ? d->k_out_stride : 0) | (d->v_out ? d->v_out_stride : 0)) & 7))
        return fail(FBLT_ERR_ARG, "%s: bf16 row strides must be multiples of 8 elements", who);
    ReadParams p;
    memset(&p, 0, sizeof(p));
    p.pv = paged_view(d->cache);
    p.rows = d->total_rows;
    p.batch = d->batch;
    p.cu = d->cu_rows;
    p.start = d->start;
    p.ko = d->k_out;
    p.vo = d->v_out;
    p.kos = d->k_out_stride;
    p.vos = d->v_out_stride;
    cudaStream_t s = (cudaStream_t)stream;
    const bool e4 = d->cache.format == FBLT_KV_E4M3;
    switch (d->cache.head_dim) {
    case 32: return e4 ? launch_read<32, FBLT_KV_E4M3>(p, bf16, s) : launch_read<32, FBLT_KV_INT8>(p, bf16, s);
    case 64: return e4 ? launch_read<64, FBLT_KV_E4M3>(p, bf16, s) : launch_read<64, FBLT_KV_INT8>(p, bf16, s);
    default: return e4 ? launch_read<128, FBLT_KV_E4M3>(p, bf16, s) : launch_read<128, FBLT_KV_INT8>(p, bf16, s);
    }
}
