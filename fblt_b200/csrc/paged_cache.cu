// Rows in and out of the 8-bit paged KV cache: per-head norm + rotation (fblt_qk_norm_rope), the same with K and V
// quantised into their pages (fblt_paged_append), and the way back (fblt_paged_read).
//
// All three are one pass over the data: head_dim / 4 lanes hold one (row, head) in registers, four values each, so the
// sum of squares and the largest magnitude are shuffles inside those lanes and nothing is read twice. What bounds
// them is HBM (reading and writing every value once), as long as a value costs few instructions: lanes keep a head and
// walk down the rows of their CTA, so that what belongs to the head (pointers, gains, the kind of work) is set up once
// and a row costs additions (with a division per value group instead, the launch was bound by instruction issue).
//
// Measured (B200): norm + rotation of a prompt's q and k, 680 MB moved: 118-121 us, 5.7 TB/s; prompts appended and read
// back 311-326 us against 223 us of bytes (K goes through 64-bit arithmetic; half of the warps fit); 1.27 GB read back from
// caches 202 us, 6.2 TB/s; one token's rows 4.7 us, a launch. The first values of every lane are asked for before the look-up
// of the rows, whose two dependent loads they hide.
#include "paged.cuh"

namespace fblt {

constexpr int kRowThreads = 256;
constexpr int kMaxRows = 8;  // rows of one CTA
constexpr int kRowLoads = 3; // rows of a head whose values a lane has in flight (64 registers and 4 CTAs an SM: 4 spill)

struct RowInfo {
    int64_t at; // row of head 0 in the pool (PagedView::row), < 0: no page
    int pos;    // < 0: the row is not to be touched
    int pad;
};

struct NormRopeParams {
    PagedView pv;     // append
    int64_t rows;
    int batch, qh, kh, rows_per_cta, rope_len, parts; // parts: log2, see split_rows
    const float *q, *k, *v;
    int64_t qs, ks, vs;
    float *qo, *ko;
    int64_t qos, kos;
    const float *qg, *kg, *cs, *sn;
    float eps;
    const int32_t *pos;          // norm + rotation alone
    const int32_t *cu, *base;    // append
};

// Sequence, position and page of packed row r, by a whole warp: the last b with cu[b] <= r is found 32 ways at a time
// (three look-ups for 32 k sequences instead of fifteen). Every lane gets the answer.
__device__ __forceinline__ RowInfo find_row(const PagedView &pv, const int32_t *cu, const int32_t *base, int batch, int total,
                                            int r, int lane) {
    RowInfo ri;
    ri.at = ri.pos = -1;
    ri.pad = 0;
    // sequences of one length: the row says which one it is; all that it needs of the sequence is asked for at once
    int lo = (int)((int64_t)r * batch / total);
    int r0 = __ldg(cu + lo), r1 = __ldg(cu + lo + 1), p0 = base ? __ldg(base + lo) : 0;
    if (r0 > r || r >= r1) {
        lo = 0;
        for (int n = batch; n > 1;) { // the answer lies in [lo, lo + n)
            const int step = (n + 31) >> 5, at = lo + lane * step;
            const bool le = lane * step < n && __ldg(cu + at) <= r;
            const int k = max(0, __popc(__ballot_sync(0xffffffffu, le)) - 1); // cu ascends: the lanes that say yes are the first ones
            lo += k * step;
            n = min(step, n - k * step);
        }
        r0 = __ldg(cu + lo), r1 = __ldg(cu + lo + 1), p0 = base ? __ldg(base + lo) : 0;
    }
    int count;
    if (!paged_seq_ok(pv, r0, r1, p0, total, count)) return ri;
    if (r < r0 || r >= r0 + count) {
        pv.raise(FBLT_PAGED_BAD_LENGTH);
        return ri;
    }
    ri.pos = p0 + (r - r0);
    const int pi = ri.pos / pv.page_size, page = pv.page(lo, pi);
    if (page < 0) pv.raise(FBLT_PAGED_BAD_PAGE);
    else ri.at = pv.row(page, 0, ri.pos - pi * pv.page_size);
    return ri;
}

// Sums and maxima over the lanes of one head; groups of a warp may be in different branches, so each names its own lanes.
template <int LANES, class T>
__device__ __forceinline__ T group_sum(uint32_t mask, T v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}
template <int LANES>
__device__ __forceinline__ float group_max(uint32_t mask, float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
}

// Four values of a lane into the codes of their row, whose exponent the group agrees on.
template <int FMT, int LANES>
__device__ __forceinline__ uint32_t quantise4(const PagedView &pv, uint32_t mask, const float (&v)[4], int &e, bool live) {
    using F = KvFormat<FMT>;
    const float top = (float)F::kQmax;
    float a = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    const float odd = fmaf(v[0], 0.0f, v[1] * 0.0f) + fmaf(v[2], 0.0f, v[3] * 0.0f); // 0, or NaN
    float w[4] = {v[0], v[1], v[2], v[3]};
    const bool bad = !(odd == 0.0f);
    if (bad) { // the exponent comes from the finite values; NaN becomes 0, an infinity the largest code
        if (live) pv.raise(FBLT_PAGED_NONFINITE);
        a = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (finite_f(w[i])) a = fmaxf(a, fabsf(w[i]));
            else if (isnan(w[i])) w[i] = 0.0f;
        }
    }
    e = F::exponent(group_max<LANES>(mask, a));
    const float s = exp2_int(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] *= s;
    if (bad || e == F::kEmax) { // elsewhere |w| <= Qmax already
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fminf(fmaxf(w[i], -top), top);
    }
    return F::codes(w[0], w[1], w[2], w[3]);
}

// The float that lies between a double's neighbours below and above it and is odd where the double is none: rounding it
// once more, to fewer bits, gives what rounding the double would have given.
__device__ __forceinline__ float round_odd(double d) {
    const float f = __double2float_rz(d);
    return (double)f == d || isnan(d) ? f : __int_as_float(__float_as_int(f) | 1);
}

// 1 / sqrt(a) to 2^-43: the single-precision estimate y (2^-22) and one step of Newton's iteration, y + y (1 - a y^2) / 2.
__device__ __forceinline__ double rsqrt_43(double a) {
    const double y = (double)rsqrtf((float)a);
    return a > 1e-30 && a < 1e30 ? fma(0.5 * y, fma(-a * y, y, 1.0), y) : rsqrt(a);
}

// FMT < 0: norm + rotation only; the heads of K and of Q. Otherwise K, V (both quantised into the pages) and Q.
// K rows that are normalised or rotated before they are quantised go through 64 bits: a code beside a border is decided
// by the last bits of fp32, and this way it is the code of the definition.
template <int HD, int FMT>
__global__ void __launch_bounds__(kRowThreads, 4) norm_rope_kernel(const NormRopeParams p) {
    constexpr int LPH = HD / 4, GROUPS = kRowThreads / LPH, U = kRowLoads;
    constexpr bool APPEND = FMT >= 0;
    __shared__ RowInfo info[kMaxRows];
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows_per_cta;
    const int nrows = (int)min((int64_t)p.rows_per_cta, p.rows - row0);
    const int units = p.qh + (APPEND ? 2 : 1) * p.kh;
    const int group = tid / LPH, lane = tid % LPH;
    const uint32_t mask = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1) << ((tid & 31) / LPH * LPH);
    const int nkv = APPEND ? 2 * p.kh : p.kh;
    // K first, then V, then Q: the long way through 64 bits runs beside the others' work, not behind it
    int kind, head;
    int64_t ss;
    const float *src;
    int row_a, row_b;
    const auto item_of = [&](int item) {
        const int unit = item >> p.parts, part = item & ((1 << p.parts) - 1), per = (p.rows_per_cta + (1 << p.parts) - 1) >> p.parts;
        row_a = min(part * per, nrows);
        row_b = min(row_a + per, nrows);
        kind = unit >= nkv ? 0 : unit < p.kh ? 1 : 2;
        head = unit - (kind == 0 ? nkv : kind == 1 ? 0 : p.kh);
        ss = kind == 0 ? p.qs : kind == 1 ? p.ks : p.vs;
        src = (kind == 0 ? p.q : kind == 1 ? p.k : p.v) + (row0 + row_a) * ss + head * HD + lane * 4;
    };
    float4 x[U];
    const auto load = [&](int r) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u < row_b) x[u] = *reinterpret_cast<const float4 *>(src + (int64_t)u * ss);
        src += (int64_t)U * ss;
    };
    const int items = units << p.parts;
    if (group < items) { // the first values travel while the rows are looked up
        item_of(group);
        load(row_a);
    }
    if (APPEND) {
        for (int r = tid >> 5; r < nrows; r += kRowThreads / 32) {
            const RowInfo ri = find_row(p.pv, p.cu, p.base, p.batch, (int)p.rows, (int)row0 + r, tid & 31);
            if ((tid & 31) == 0) {
                info[r] = ri;
                if (p.cs && ri.pos >= p.rope_len) p.pv.raise(FBLT_PAGED_BAD_POSITION);
            }
        }
    } else if (tid < nrows) {
        RowInfo ri;
        ri.pos = p.pos ? p.pos[row0 + tid] : 0;
        ri.at = ri.pad = 0;
        info[tid] = ri;
        if (p.cs && (ri.pos < 0 || ri.pos >= p.rope_len)) p.pv.raise(FBLT_PAGED_BAD_POSITION);
    }
    __syncthreads();
    const float2 *cs = reinterpret_cast<const float2 *>(p.cs) + lane, *sn = reinterpret_cast<const float2 *>(p.sn) + lane;
    float2 c[U], s[U];
    const auto load_rope = [&](int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r + u >= row_b) break;
            const int pos = info[r + u].pos;
            if (p.cs && (unsigned)pos < (unsigned)p.rope_len) {
                c[u] = __ldg(cs + (int64_t)pos * (HD / 4));
                s[u] = __ldg(sn + (int64_t)pos * (HD / 4));
            }
        }
    };
    for (int item = group; item < items; item += GROUPS) {
        if (item != group) {
            item_of(item);
            load(row_a);
        }
        if (!APPEND || kind == 0) {
            const int64_t ds = kind == 0 ? p.qos : p.kos;
            float *dst = (kind == 0 ? p.qo : p.ko) + (row0 + row_a) * ds + head * HD + lane * 4;
            const float *gain = kind == 0 ? p.qg : p.kg;
            const float4 g = gain ? __ldg(reinterpret_cast<const float4 *>(gain) + lane) : make_float4(1.f, 1.f, 1.f, 1.f);
            for (int r = row_a; r < row_b; r += U) {
                if (r > row_a) load(r);
                load_rope(r);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (r + u >= row_b) break;
                    const int pos = info[r + u].pos;
                    if (gain) {
                        const float sum = group_sum<LPH>(mask, x[u].x * x[u].x + x[u].y * x[u].y + (x[u].z * x[u].z + x[u].w * x[u].w));
                        const float inv = rsqrtf(fmaf(sum, 1.0f / HD, p.eps));
                        x[u] = make_float4(x[u].x * (inv * g.x), x[u].y * (inv * g.y), x[u].z * (inv * g.z), x[u].w * (inv * g.w));
                    }
                    if (p.cs && (unsigned)pos < (unsigned)p.rope_len) {
                        rope_rotate(x[u].x, x[u].y, c[u].x, s[u].x);
                        rope_rotate(x[u].z, x[u].w, c[u].y, s[u].y);
                    }
                    if (!APPEND || pos >= 0) *reinterpret_cast<float4 *>(dst + (int64_t)u * ds) = x[u];
                }
                dst += (int64_t)U * ds;
            }
        }
        if constexpr (APPEND) {
            if (kind == 0) continue;
            uint8_t *codes = (kind == 1 ? p.pv.kc : p.pv.vc) + lane * 4;
            int8_t *exps = kind == 1 ? p.pv.ke : p.pv.ve;
            const int64_t skip = (int64_t)head * p.pv.page_size; // from head 0's row of a page to this head's
            const bool norm = kind == 1 && p.kg, rope = kind == 1 && p.cs;
            float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
            if (norm) g = __ldg(reinterpret_cast<const float4 *>(p.kg) + lane);
            for (int r = row_a; r < row_b; r += U) {
                if (r > row_a) load(r);
                if (rope) load_rope(r);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (r + u >= row_b) break;
                    const RowInfo ri = info[r + u];
                    float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                    if (norm || rope) {
                        double d[4] = {v[0], v[1], v[2], v[3]};
                        if (norm) {
                            const double sum = group_sum<LPH>(mask, d[0] * d[0] + d[1] * d[1] + (d[2] * d[2] + d[3] * d[3]));
                            const double inv = rsqrt_43(sum * (1.0 / HD) + (double)p.eps);
                            d[0] *= inv * (double)g.x, d[1] *= inv * (double)g.y, d[2] *= inv * (double)g.z, d[3] *= inv * (double)g.w;
                        }
                        if (rope && (unsigned)ri.pos < (unsigned)p.rope_len) {
                            const double a = d[0], b = d[2];
                            d[0] = a * (double)c[u].x - d[1] * (double)s[u].x;
                            d[1] = d[1] * (double)c[u].x + a * (double)s[u].x;
                            d[2] = b * (double)c[u].y - d[3] * (double)s[u].y;
                            d[3] = d[3] * (double)c[u].y + b * (double)s[u].y;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = round_odd(d[i]);
                    }
                    int e;
                    const uint32_t w = quantise4<FMT, LPH>(p.pv, mask, v, e, ri.pos >= 0);
                    if (ri.at >= 0) {
                        const int64_t at = ri.at + skip;
                        *reinterpret_cast<uint32_t *>(codes + at * HD) = w;
                        if (lane == 0) exps[at] = (int8_t)e;
                    }
                }
            }
        }
    }
}

struct ReadParams {
    PagedView pv;
    int rows, batch, rows_per_cta, parts;
    const int32_t *cu, *start;
    void *ko, *vo;
    int64_t kos, vos;
};

template <int HD, int FMT, bool BF16>
__global__ void __launch_bounds__(kRowThreads) paged_read_kernel(const ReadParams p) {
    constexpr int LPH = HD / 4, GROUPS = kRowThreads / LPH, U = 8;
    __shared__ RowInfo info[kMaxRows];
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows_per_cta;
    const int nrows = (int)min((int64_t)p.rows_per_cta, p.rows - row0);
    for (int r = tid >> 5; r < nrows; r += kRowThreads / 32) {
        const RowInfo ri = find_row(p.pv, p.cu, p.start, p.batch, p.rows, (int)row0 + r, tid & 31);
        if ((tid & 31) == 0) info[r] = ri;
    }
    __syncthreads();
    const int kh = p.pv.kvh, units = (p.ko && p.vo ? 2 : 1) * kh, group = tid / LPH, lane = tid % LPH;
    const int items = units << p.parts, per = (p.rows_per_cta + (1 << p.parts) - 1) >> p.parts;
    for (int item = group; item < items; item += GROUPS) {
        const int unit = item >> p.parts, row_a = (item & ((1 << p.parts) - 1)) * per, row_b = min(row_a + per, nrows);
        const bool is_v = !p.ko || unit >= kh;
        const int head = unit >= kh ? unit - kh : unit;
        const int64_t skip = (int64_t)head * p.pv.page_size, ds = is_v ? p.vos : p.kos;
        const uint8_t *codes = (is_v ? p.pv.vc : p.pv.kc) + skip * HD + lane * 4;
        const int8_t *exps = (is_v ? p.pv.ve : p.pv.ke) + skip;
        int64_t to = (row0 + row_a) * ds + head * HD + lane * 4;
        void *dst = is_v ? p.vo : p.ko;
        for (int r = row_a; r < row_b; r += U) {
            uint32_t w[U];
            int e[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + u >= row_b) break;
                const int64_t at = info[r + u].at;
                w[u] = 0;
                e[u] = 0;
                if (at >= 0) {
                    w[u] = *reinterpret_cast<const uint32_t *>(codes + at * HD);
                    e[u] = exps[at];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + u >= row_b) break;
                if (info[r + u].pos < 0) continue;
                const float4 x = kv_values<FMT>(w[u], kv_scale<FMT>(e[u]));
                if (BF16) {
                    const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
                    uint2 o;
                    o.x = *reinterpret_cast<const uint32_t *>(&lo);
                    o.y = *reinterpret_cast<const uint32_t *>(&hi);
                    *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(dst) + to + (int64_t)u * ds) = o;
                } else {
                    *reinterpret_cast<float4 *>(static_cast<float *>(dst) + to + (int64_t)u * ds) = x;
                }
            }
            to += (int64_t)U * ds;
        }
    }
}

// Rows of one CTA: one while that fills the GPU, more when the launch is long anyway: the row look-up is then shared,
// and a row's loads overlap the others' (in whole batches of `loads`, since a last, short batch waits as long as a full one).
// Norm and append, 4 CTAs an SM: 4 rows of 2048 sequences 40 us at 6 rows a CTA, 49 us at 3; prompts (30 k rows appended and
// read back) 314 us at 6 rows, 328 us at 12; norm alone (16 k rows) 118 us at 6, 127 us at 12. Reading, 8 CTAs an SM: 204 us
// at 8 rows, 232 us at 4, 210 us at 16.
static int rows_per_cta(int64_t rows, int64_t ctas, int loads, int most) {
    const int64_t r = rows / ctas;
    if (r < loads) return r < 1 ? 1 : (int)r;
    return (r > most ? most : (int)r) / loads * loads;
}

// A CTA's groups share `units` heads x `rows` rows in items of one head and 1 / 2^parts of the rows: the split whose
// busiest group has the fewest rows.
static int split_rows(int units, int rows, int groups) {
    int best = 0, least = INT_MAX;
    for (int lp = 0; lp == 0 || (1 << lp) <= rows; ++lp) {
        const int64_t rounds = (((int64_t)units << lp) + groups - 1) / groups, per = (rows + (1 << lp) - 1) >> lp;
        if (rounds * per < least) least = (int)(rounds * per), best = lp;
    }
    return best;
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
    p.rows_per_cta = rows_per_cta(p.rows, kPlanSms * 8, kRowLoads, 2 * kRowLoads);
    p.parts = split_rows(p.qh + (FMT < 0 ? 1 : 2) * p.kh, p.rows_per_cta, kRowThreads / (HD / 4));
    const int64_t grid = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
    if (grid > INT_MAX) return fail(FBLT_ERR_LIMIT, "%s: too many rows", what);
    norm_rope_kernel<HD, FMT><<<(unsigned)grid, kRowThreads, 0, s>>>(p);
    count_launch();
    return check_launch(what);
}

template <int HD, int FMT>
static int launch_read(ReadParams &p, bool bf16, cudaStream_t s) {
    p.rows_per_cta = rows_per_cta(p.rows, kPlanSms * 4, 1, 8);
    p.parts = split_rows((p.ko && p.vo ? 2 : 1) * p.pv.kvh, p.rows_per_cta, kRowThreads / (HD / 4));
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
