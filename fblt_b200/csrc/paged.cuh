// The 8-bit paged KV cache as the kernels see it: page lookup with bounds, the code <-> value
// conversions and the checks every host entry point makes of the cache description.
#pragma once

#include "common.cuh"
#include "tc5.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <atomic>
#include <limits.h>
#include <string.h>

namespace fblt {

constexpr int kPlanSms = 148; // SMs of a B200, which the plans are made for

struct PagedView {
    uint8_t *kc, *vc;
    int8_t *ke, *ve;
    const int32_t *table;
    int64_t table_stride;
    int num_pages, max_pages, page_size, kvh;
    int32_t *status;

    __device__ __forceinline__ void raise(int bit) const {
        if (status) atomicOr(status, bit);
    }
    // Page that holds entry `pi` of sequence b's table, -1 if there is none.
    __device__ __forceinline__ int page(int b, int pi) const {
        if (pi >= max_pages) return -1;
        const int id = __ldg(table + (int64_t)b * table_stride + pi);
        return (unsigned)id < (unsigned)num_pages ? id : -1;
    }
    // Row index of (page, kv head, slot): element offset of its exponent; times head_dim that of its codes.
    __device__ __forceinline__ int64_t row(int page, int head, int slot) const {
        return ((int64_t)page * kvh + head) * page_size + slot;
    }
};

inline PagedView paged_view(const fblt_paged_cache &c) {
    PagedView v;
    v.kc = c.k_codes;
    v.vc = c.v_codes;
    v.ke = c.k_exp;
    v.ve = c.v_exp;
    v.table = c.page_table;
    v.table_stride = c.page_table_stride;
    v.num_pages = c.num_pages;
    v.max_pages = c.max_pages;
    v.page_size = c.page_size;
    v.kvh = c.num_kv_heads;
    v.status = c.status;
    return v;
}

// Raises a kernel's dynamic shared memory limit on the current device, once (the call costs a microsecond of a decode
// step). `done`: a bit per device ordinal; devices past 63 are set every time.
inline int allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    FBLT_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit & done.load(std::memory_order_relaxed)) return FBLT_OK;
    FBLT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return FBLT_OK;
}

int validate_paged_cache(const fblt_paged_cache &c, int batch, const char *who); // paged_cache.cu

// New rows of a sequence: packed rows [r0, r1), first position base; n of them. False (and the status bit) where that is
// not a sequence.
__device__ __forceinline__ bool paged_seq_ok(const PagedView &pv, int r0, int r1, int base, int total, int &n) {
    n = r1 - r0;
    if (r0 < 0 || r1 < r0 || r1 > total || base < 0 || base > INT_MAX - n) {
        pv.raise(FBLT_PAGED_BAD_LENGTH);
        n = 0;
        return false;
    }
    return true;
}
// The same for sequence b of the tables.
__device__ __forceinline__ bool paged_seq(const PagedView &pv, const int32_t *cu, const int32_t *base_len, int total, int b,
                                          int &r0, int &n, int &base) {
    r0 = cu[b];
    base = base_len ? base_len[b] : 0;
    return paged_seq_ok(pv, r0, cu[b + 1], base, total, n);
}

// 2^e as a float, -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }
// The same for any e <= 127, below 2^-149 zero.
__device__ __forceinline__ float exp2_low(int e) { return e >= -126 ? exp2_int(e) : e < -149 ? 0.0f : __int_as_float(1 << (e + 149)); }

// Scales of V within a stage or tile, 2^(e - et) with et the largest, span 247 powers of two, the mask may take the largest
// ones out of a row's sum, and p 2^(e - et) has to be a float for every p up to 2^4: they are kept 2^kVUp higher.
constexpr int kVUp = 123, kVSpan = 247;

template <int FMT>
struct KvFormat;

// e4m3: sign, 4 exponent bits (bias 7), 3 mantissa bits.
template <>
struct KvFormat<FBLT_KV_E4M3> {
    static constexpr int kEmin = -117, kEmax = 119, kQmax = 448;
    // least e with a <= 448 * 2^e, from the bits of a = 1.m * 2^x: x - 8, one more where the significand passes 1.75
    static __device__ __forceinline__ int exponent(float a) {
        const int b = __float_as_int(a);
        const int e = (b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
        return min(max(e, kEmin), kEmax);
    }
    // four codes (one word) -> halves of codes 0, 1 and of codes 2, 3
    static __device__ __forceinline__ void halves(uint32_t w, uint32_t &h01, uint32_t &h23) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(h01), "=r"(h23)
            : "r"(w));
    }
    // four scaled finite values -> one word of codes
    static __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
};

template <>
struct KvFormat<FBLT_KV_INT8> {
    static constexpr int kEmin = -126, kEmax = 121, kQmax = 127;
    // least e with a <= 127 * 2^e: x - 6, one more where the significand passes 127 / 64
    static __device__ __forceinline__ int exponent(float a) {
        const int b = __float_as_int(a);
        const int e = (b >> 23) - 127 - 6 + ((b & 0x7fffff) > 0x7e0000 ? 1 : 0);
        return min(max(e, kEmin), kEmax);
    }
    // byte ^ 0x80 below the exponent of 1024 is the half 1024 + 128 + code: exact, and so is the difference
    static __device__ __forceinline__ void halves(uint32_t w, uint32_t &h01, uint32_t &h23) {
        w ^= 0x80808080u;
        const __half2 off = __float2half2_rn(1152.0f);
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off), y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
        h01 = *reinterpret_cast<const uint32_t *>(&x);
        h23 = *reinterpret_cast<const uint32_t *>(&y);
    }
    static __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) {
        // 1.5 * 2^23 + x rounds x to the nearest integer, ties to even, and has it in its low bits
        const float o = 12582912.0f;
        const uint32_t i = __byte_perm(__float_as_uint(a + o), __float_as_uint(b + o), 0x0040);
        const uint32_t j = __byte_perm(__float_as_uint(c + o), __float_as_uint(d + o), 0x0040);
        return __byte_perm(i, j, 0x5410);
    }
};

// Four codes of one word -> their values, `s` = 2^e.
template <int FMT>
__device__ __forceinline__ float4 kv_values(uint32_t w, float s) {
    uint32_t a, b;
    KvFormat<FMT>::halves(w, a, b);
    const float2 x = __half22float2(*reinterpret_cast<__half2 *>(&a)), y = __half22float2(*reinterpret_cast<__half2 *>(&b));
    return make_float4(x.x * s, x.y * s, y.x * s, y.y * s);
}
template <int FMT>
__device__ __forceinline__ float kv_scale(int e) { // exponents outside the format's range are not written by the library
    return exp2_int(min(max(e, KvFormat<FMT>::kEmin), KvFormat<FMT>::kEmax));
}

// x, y -> (hi, lo) planes of two halves each: 22 bits of a value of ordinary size
__device__ __forceinline__ void split_half2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// A bounded wait of a whole warp, with one answer: lanes that gave up alone would leave the others' shuffles without partners.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, const volatile int *abort_word) {
    return __all_sync(0xffffffffu, mbar_wait_abort(bar, parity, abort_word));
}

// What the attention kernels get. The rows of one kv head are numbered r = i * G + g: head kvh * G + g of token i.
struct PagedAttnParams {
    PagedView pv;
    int batch, H, G, total, max_new, block_mode, window, splits, row_tiles;
    const int32_t *cu, *base;
    const float *q;
    int64_t qs;
    float *out;
    int64_t os;
    float *ws;
    float qscale; // scale * log2(e)
};

// A CTA's place: kv heads of a piece side by side, then the pieces, then (sequence, tile of rows) -- in one dimension of the
// grid, whose other two end at 65535.
struct PagedCtaAt {
    int kvh, split, unit;
};
__device__ __forceinline__ PagedCtaAt paged_cta(const PagedAttnParams &p) {
    PagedCtaAt at;
    const unsigned r = blockIdx.x / (unsigned)p.pv.kvh;
    at.kvh = (int)(blockIdx.x - r * (unsigned)p.pv.kvh);
    at.unit = (int)(r / (unsigned)p.splits);
    at.split = (int)(r - (unsigned)at.unit * (unsigned)p.splits);
    return at;
}
inline unsigned paged_grid(const PagedAttnParams &p) { // paged_plan_check: fits
    return (unsigned)((int64_t)p.pv.kvh * p.splits * p.batch * p.row_tiles);
}

// Keys that rows [row0, row0 + rows) of a sequence with n new rows at `base` see between them. Positions beyond the page
// table hold no key, and however large a length is, nothing walks past them (nor past where a stage's last key would leave
// 32 bits).
struct RowRange {
    int lo, hi; // keys the tile's rows see between them
};
__device__ __forceinline__ RowRange tile_range(const PagedAttnParams &p, int base, int n, int row0, int rows) {
    RowRange r;
    const int i0 = row0 / p.G, i1 = min(n - 1, (row0 + rows - 1) / p.G);
    r.hi = p.block_mode ? base + n : base + i1 + 1;
    r.lo = !p.block_mode && p.window > 0 ? max(0, base + i0 - p.window + 1) : 0;
    const int64_t room = (int64_t)p.pv.max_pages * p.pv.page_size;
    const int cap = room < INT_MAX - 4096 ? (int)room : (INT_MAX - 4096) & ~15;
    if (r.hi > cap) {
        p.pv.raise(FBLT_PAGED_BAD_PAGE);
        r.hi = cap;
    }
    r.lo = min(r.lo, r.hi);
    return r;
}

} // namespace fblt
