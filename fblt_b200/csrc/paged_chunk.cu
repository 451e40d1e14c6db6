// Attention of a chunk of new rows over the 8-bit paged KV cache on tcgen05 (fblt_paged_attn with many query rows per
// kv head: prompts taken in chunks).
//
// CTA = (sequence, kv head, key range, 256 query rows as two tiles of 128), one per SM; K and V tiles of BN keys are
// converted once for both query tiles. An 8-bit code is a half as it stands, so K and V are ONE fp16 plane each and the
// 22 bits of fp32 class come from two planes of Q and of P: two MMAs where 16-bit attention has one.
// The exponents of a tile's K (V) go into its halves, relative to the tile's largest, where they lie within 2^4 of each
// other (rows of one head: nearly always); otherwise they multiply the columns of S (P).
//   S = Q K^T    Q is scaled by its row's power of two.
//   O += P V     2^et is the largest scale of the tile's V. O is in units of
//                2^R, a row's own R, which follows the largest p 2^et the row has had, so that P's halves keep the 22
//                bits of what counts; et, R and the maximum meet in the exponent of 2^x and cost nothing per score.
//
// Roles (13 warps at work), which meet on mbarriers only; every wait is bounded:
//   softmax (2 x 4 warps)  one thread per query row (TMEM lane): running maximum and sum, P back to TMEM over the scores
//                          it came from. O stays in TMEM and is rescaled only where a maximum has grown by more than 2^4.
//   converters (4 warps)   pages -> registers (one tile ahead) -> halves in shared memory, in 8-row x 16-byte core
//                          matrices (K read K-major, V MN-major: the same bytes, no transposition)
//   issuer (1 warp)        while one query tile's softmax runs, the tensor cores have the other tile's products
// Q's planes are TMEM operands (head_dim 128: the first one; the other stays in shared memory).
//
// Measured (B200): 2048 new rows x 16 heads, head_dim 64, behind 31 k keys: 632-650 us, 405 TFLOP/s of the formula's
// products and twice that on the tensor cores (two planes); ragged chunks at head_dim 128: 315-330 us. What bounds it is
// the chain of one query tile: a step of 128 keys takes 4960 cycles, of which its 512 exponentials a scheduler 2150
// (8 cycles a warp instruction), the wait for P V and the next S 1250, reading scores and their maximum 470, rescaling 450,
// folding 330 (head_dim 128, whose sums fold into output rows: 850). Issue slots are 43 %, tensor cores 34 % busy (small
// case). Measured and slower: three bf16 planes of P 757 us; S beside P instead of under it, tiles of 96 keys 715 us;
// two threads a row 704 us; the query tiles in turns 695 us; a share of the exponentials as polynomials 649-698 us.
#include "paged.cuh"

namespace fblt {

constexpr int kPcThreads = 512, kPcSoft = 256, kPcConv = 128; // + the issuer's warpgroup
constexpr int kPcRows = 128;

__device__ unsigned int g_chunk_error; // 0 = ok; otherwise (code << 24) | blockIdx.x of the first CTA that gave up

template <int HD>
struct PcShape {
    static constexpr int BN = HD == 128 ? 64 : 128; // keys of a tile: S, P and O of two query tiles fit 512 columns
    static constexpr int kQPlane = HD == 128 ? kPcRows * HD * 2 : 0, kKv = BN * HD * 2;
    static constexpr int kOffKv = 2 * kQPlane; // head_dim 128: the second plane of Q of both tiles
    static constexpr int kOffSum = kOffKv + 4 * kKv; // head_dim 32, 64: folded sums, see the softmax
    // (and, before and after the loop, rows on their way between memory and the threads: 4 KB a warp, Q's planes whole)
    static constexpr int kSmem = kOffSum + 2 * kPcRows * (HD == 128 ? 64 : HD) * 4;
    // TMEM columns of a query tile: S / P, O; behind both tiles the planes of Q
    static constexpr int kO = BN, kTile = BN + HD, kQCols = HD / 2, kQTile = HD == 128 ? kQCols : 2 * kQCols, kQ = 2 * kTile;
    static_assert(kQ + 2 * kQTile <= 512, "TMEM");
};
constexpr int kPcHead = 10;   // P in units of 2^(R - kPcHead), R at most 4 below the largest exponent: halves up to 2^15
constexpr int kPcFold = 512;  // keys whose products the tensor cores sum: they cut every sum off below 24 bits, which pulls
                              // O towards zero by about 2e-8 an MMA (9e-6 over 31 k keys in eight pieces; 512 keys are 64
                              // MMAs); what they have is then added, rounded, to sums of its own
constexpr int kPcNarrow = 4;  // exponents of a tile go into its halves where they lie this close

// fp16 operands, fp32 accumulate; B K-major or MN-major
__host__ __device__ constexpr uint32_t pc_idesc(int n, bool mn_major) {
    return (1u << 4) | ((mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kPcRows >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}

// One lane of a converged warp. The compiler knows such a branch to be the work of one thread of a uniform warp, so the
// descriptors of the products below stay in uniform registers; behind `lane == 0` each product first moves its operands
// there, which took the issuer about 90 cycles an MMA.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// Barrier of the four converter warps that tells all of them whether any has failed.
__device__ __forceinline__ bool converters_or(bool x) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any)
                 : "r"((uint32_t)x)
                 : "memory");
    return any != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

struct PcBars {
    uint64_t q_full, kv_full[2], kv_empty[2], s_full[2], p_ready[2], o_full, fin;
};

template <int HD, int FMT>
__global__ void __launch_bounds__(kPcThreads, 1) paged_chunk_kernel(const PagedAttnParams p) {
    using F = KvFormat<FMT>;
    using S = PcShape<HD>;
    constexpr int BN = S::BN, CH = BN / 32, PR = HD + 4, kFold = kPcFold / BN;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ PcBars bars;
    __shared__ __align__(16) float vscale[2][BN];
    __shared__ int kunder[2][BN]; // a key's exponent below the tile's largest
    __shared__ __align__(16) int top_of[2][4]; // largest exponent of the tile's K, of its V; whether each is too wide for its halves
    __shared__ int4 range[2][4];
    __shared__ __align__(8) uint8_t present[2][8]; // groups of 16 keys whose page exists and that the CTA reads
    __shared__ int q_exp[2][kPcRows]; // power of two of a query row; + 4096 where a value of it is not finite
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort;
    const volatile int *abortp = &s_abort;

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const PagedCtaAt at = paged_cta(p);
    const int kvh = at.kvh, split = at.split, b = at.unit / p.row_tiles;
    const int rt = p.row_tiles - 1 - (at.unit - b * p.row_tiles); // later rows see more keys: they go first
    int r0, n, base;
    if (!paged_seq(p.pv, p.cu, p.base, p.total, b, r0, n, base)) return;
    if (n > p.max_new && tid == 0) p.pv.raise(FBLT_PAGED_BAD_LENGTH);
    const int rows = min(n, p.max_new) * p.G, row0 = rt * 2 * kPcRows;
    if (row0 >= rows) return;
    const int tiles = rows - row0 > kPcRows ? 2 : 1;
    const RowRange rr = tile_range(p, base, n, row0, min(2 * kPcRows, rows - row0));
    const int first = rr.lo & ~15, steps = (rr.hi - first + BN - 1) / BN, per = (steps + p.splits - 1) / p.splits;
    const int st0 = min(steps, split * per), nst = min(steps, st0 + per) - st0;
    const int kb0 = first + st0 * BN;
    const uint32_t sbase = smem_u32(smem);
    // A piece without a key: zeros, of weight 0 where pieces are merged. It is left before anything is staged: the products,
    // which order a warp's use of the shared memory that another one's query rows came through, are what such a piece lacks.
    if (nst == 0) {
        const int here = min(2 * kPcRows, rows - row0);
        for (int it = tid; it < here * (HD / 4); it += kPcThreads) {
            const int r = row0 + it / (HD / 4), d = it % (HD / 4) * 4, i = r / p.G, head = kvh * p.G + (r - i * p.G);
            float *dst = p.splits > 1 ? p.ws + (((int64_t)(r0 + i) * p.H + head) * p.splits + split) * PR
                                      : p.out + (int64_t)(r0 + i) * p.os + (int64_t)head * HD;
            *reinterpret_cast<float4 *>(dst + d) = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p.splits > 1 && d == 0) *reinterpret_cast<float2 *>(dst + HD) = make_float2(-INFINITY, 0.0f);
        }
        return;
    }

    auto give_up = [&](unsigned code) {
        *(volatile int *)&s_abort = 1;
        atomicCAS(&g_chunk_error, 0u, (code << 24) | (blockIdx.x & 0xffffffu));
    };

    if (tid == 0) {
        mbar_init(&bars.q_full, tiles * kPcRows);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.kv_full[i], kPcConv);
            mbar_init(&bars.kv_empty[i], 1);
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_ready[i], kPcRows);
        }
        mbar_init(&bars.o_full, 1);
        mbar_init(&bars.fin, 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // Registers follow the roles: 256 x 200 + 128 x 72 + 128 x 40 = the 512 x 128 of the launch.
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ================= softmax: this thread's query row =================
        const int T = warp >> 2, rl = (warp & 3) * 32 + lane, r = row0 + T * kPcRows + rl;
        if (T < tiles) {
            const bool live = r < rows;
            const int rc = min(r, rows - 1), i = rc / p.G, head = kvh * p.G + (rc - i * p.G), pos = base + i;
            const int hi = p.block_mode ? base + n : pos + 1;
            const int lo = !p.block_mode && p.window > 0 ? max(0, pos - p.window + 1) : 0;
            const int span = hi - lo;
            const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T * S::kTile;
            // ---- query planes: q scale log2(e) 2^e with the row's largest value in [2^13, 2^14). Rows come in whole (HD / 4
            // lanes each; a thread that read its own row took 20 to 40 thousand clocks), the planes go through shared
            // memory to the threads that own them, 16-byte units exchanged within a row so that columns are free of conflicts.
            int qe; // the row of Q was multiplied by 2^qe
            bool qbad; // a query value that is not finite
            {
                constexpr int LPR = HD / 4, RPI = 32 / LPR, UNITS = HD / 8, B = HD == 32 ? 8 : 16; // lanes a row, rows an instruction, units a row
                const uint64_t own = (uint64_t)(p.q + (int64_t)(r0 + i) * p.qs + (int64_t)head * HD);
                uint8_t *hold = smem + S::kOffSum + T * kPcRows * (HD == 128 ? 64 : HD) * 4; // first plane, then (HD <= 64) the second
                const int q4 = lane % LPR;
#pragma unroll 1
                for (int it = 0; it < 32 / RPI; it += B) {
                    float4 v[B];
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        const uint64_t row = __shfl_sync(0xffffffffu, own, (it + k) * RPI + lane / LPR);
                        v[k] = reinterpret_cast<const float4 *>(row)[q4];
                    }
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        const int row = (warp & 3) * 32 + (it + k) * RPI + lane / LPR;
                        const float w[4] = {v[k].x * p.qscale, v[k].y * p.qscale, v[k].z * p.qscale, v[k].w * p.qscale};
                        float a = 0.0f;
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (finite_f(w[e])) a = fmaxf(a, fabsf(w[e]));
                            else odd = true;
                        }
#pragma unroll
                        for (int o = LPR / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
                        const uint32_t odds = __ballot_sync(0xffffffffu, odd);
                        const int e = min(13 - ((__float_as_int(a) >> 23) - 127), 126);
                        const float up = exp2_int(e);
                        uint2 h, l;
                        split_half2(w[0] * up, w[1] * up, h.x, l.x);
                        split_half2(w[2] * up, w[3] * up, h.y, l.y);
                        const int at = row * (HD * 2) + (((q4 >> 1) ^ (row & 7 & (UNITS - 1))) * 16) + (q4 & 1) * 8;
                        *reinterpret_cast<uint2 *>(hold + at) = h;
                        if (HD == 128) // K-major core matrices
                            *reinterpret_cast<uint2 *>(smem + T * S::kQPlane + (q4 >> 1) * (kPcRows * 16) + row * 16 + (q4 & 1) * 8) = l;
                        else
                            *reinterpret_cast<uint2 *>(hold + kPcRows * HD * 2 + at) = l;
                        if (q4 == 0) q_exp[T][row] = e + ((odds >> (lane / LPR * LPR)) & (LPR == 32 ? 0xffffffffu : (1u << (LPR & 31)) - 1) ? 4096 : 0);
                    }
                }
                __syncwarp();
                qbad = q_exp[T][rl] > 2048;
                qe = q_exp[T][rl] - (qbad ? 4096 : 0);
                const uint32_t tq = tmem + ((uint32_t)((warp & 3) * 32) << 16) + S::kQ + T * S::kQTile;
#pragma unroll
                for (int pl = 0; pl < (HD == 128 ? 1 : 2); ++pl)
#pragma unroll
                    for (int c = 0; c < UNITS / 4; ++c) {
                        uint32_t x[16];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(hold + pl * (kPcRows * HD * 2) + rl * (HD * 2) +
                                                                             (((4 * c + k) ^ (rl & 7 & (UNITS - 1))) * 16));
                            x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
                        }
                        tmem_st16(tq + pl * S::kQCols + c * 16, x);
                    }
                tc_wait_st();
                tc_fence_before();
                fence_async_smem();
                mbar_arrive(&bars.q_full);
            }
            float *dst = p.splits > 1 ? p.ws + (((int64_t)(r0 + i) * p.H + head) * p.splits + split) * PR
                                      : p.out + (int64_t)(r0 + i) * p.os + (int64_t)head * HD;
            // Sums that were folded (`since`: how far O's unit has moved from theirs) lie in shared memory, a thread's next to
            // its neighbours'. At head_dim 128 there is no room for them: they lie in the warp's 32 output rows, in an order
            // of their own, lane l's k-th four values at row 4 (k % 8) + l / 8, column 32 (k / 8) + 4 (l % 8), so that an
            // access is four whole lines; a warp with fewer rows uses each row for itself.
            const bool full = __all_sync(0xffffffffu, live);
            float since = 1.0f;
            auto place = [&](int k) -> float4 * {
                if (HD <= 64) return reinterpret_cast<float4 *>(smem + S::kOffSum) + (T * (HD / 4) + k) * kPcRows + rl;
                const uint64_t row = __shfl_sync(0xffffffffu, (uint64_t)dst, 4 * (k & 7) + (lane >> 3));
                return full ? reinterpret_cast<float4 *>(row) + 8 * (k >> 3) + (lane & 7) : reinterpret_cast<float4 *>(dst) + k;
            };
            float m = -INFINITY, l = 0.0f;
            int R = 0;
            // A lane whose wait has run out goes on with the others, without waiting, and nothing is written in the end: leaving
            // alone it would take the partner of their shuffles away (and a vote on every wait costs 5 %).
            unsigned lost = 0; // which wait
            auto wait = [&](uint64_t *bar, uint32_t parity, unsigned code) {
                if (lost || mbar_wait_abort(bar, parity, abortp)) return;
                *(volatile int *)&s_abort = 1;
                lost = code;
            };
            wait(&bars.kv_full[0], 0, 0x55);
            for (int j = 0; j < nst; ++j) { // the tile's scales are there: waited for at the end of the step before
                const int st = j & 1, kb = kb0 + j * BN;
                wait(&bars.s_full[T], j & 1, 0x51);
                tc_fence_after();
                if (j > 0 && j % kFold == 0) { // O is complete: S came behind it
                    constexpr int W = HD == 128 ? 16 : 8; // fours of columns whose sums are read together
#pragma unroll 1
                    for (int c = 0; c < HD / 4; c += W) {
                        float4 v[W];
#pragma unroll
                        for (int k = 0; k < W; ++k) {
                            const float4 *at = place(c + k);
                            v[k] = j > kFold && (live || HD <= 64) ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
#pragma unroll
                        for (int h = 0; h < W; h += 8) {
                            float o[32];
                            tmem_ld32(trow + S::kO + (c + h) * 4, o);
                            tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                float4 *at = place(c + h + k);
                                if (live || HD <= 64)
                                    *at = make_float4(fmaf(v[h + k].x, since, o[4 * k]), fmaf(v[h + k].y, since, o[4 * k + 1]),
                                                      fmaf(v[h + k].z, since, o[4 * k + 2]), fmaf(v[h + k].w, since, o[4 * k + 3]));
                            }
                        }
                    }
                    since = 1.0f;
                }
                bool all = true;
#pragma unroll
                for (int g = 0; g < BN / 16; ++g) all &= present[st][g] != 0;
                const bool masked = !__all_sync(0xffffffffu, all && kb >= lo && kb + BN <= hi);
                // ---- the row's scores times K's scales, all in registers, and their maximum
                float2 y[CH][16];
                {
                    float v[CH][32];
#pragma unroll
                    for (int c = 0; c < CH; ++c) tmem_ld32(trow + c * 32, v[c]);
                    tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[c][k] = make_float2(v[c][2 * k], v[c][2 * k + 1]);
                }
                float peak[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        peak[k & 2] = max3(peak[k & 2], y[c][k].x, y[c][k].y);
                        peak[(k & 2) + 1] = max3(peak[(k & 2) + 1], y[c][k + 1].x, y[c][k + 1].y);
                    }
                const int4 tops = *reinterpret_cast<const int4 *>(top_of[st]);
                const int sc = tops.x - qe; // a score is y 2^sc
                float down = exp2_int(min(max(sc, -126), 126));
                float mx = fmaxf(fmaxf(peak[0], peak[1]), fmaxf(peak[2], peak[3])) * down;
                // Sums of 8-bit codes times query planes below 2^14 stay far from overflow, so a score is not finite only
                // where the query row is not, or where the scales took it past fp32's range (-inf weighs 0 by itself).
                if (__any_sync(0xffffffffu, masked || tops.z || qbad || sc > 126 || !(mx < INFINITY))) {
                    // where one float does not hold the scales, they are taken key by key in two
                    const bool apart = __any_sync(0xffffffffu, tops.z || sc > 126);
                    if (apart) down = 1.0f;
                    mx = -INFINITY;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const int d = kb + c * 32 + 2 * k - lo;
                            const bool there = present[st][c * 2 + k / 8] != 0;
                            if (apart) {
                                const int ex = sc - (tops.z ? kunder[st][c * 32 + 2 * k] : 0), ey = sc - (tops.z ? kunder[st][c * 32 + 2 * k + 1] : 0);
                                y[c][k].x = y[c][k].x * exp2_int(min(max(ex, -126), 126)) * exp2_int(min(max(ex, 126) - 126, 127));
                                y[c][k].y = y[c][k].y * exp2_int(min(max(ey, -126), 126)) * exp2_int(min(max(ey, 126) - 126, 127));
                            }
                            y[c][k].x = there && (unsigned)d < (unsigned)span && finite_f(y[c][k].x * down) ? y[c][k].x : -INFINITY;
                            y[c][k].y = there && (unsigned)(d + 1) < (unsigned)span && finite_f(y[c][k].y * down) ? y[c][k].y : -INFINITY;
                            mx = fmaxf(fmaxf(mx, y[c][k].x), y[c][k].y);
                        }
                    mx *= down;
                }
                // ---- O and its unit follow the maximum only when that has grown by more than 2^4 (weights exceed 1 until then),
                // and the unit alone where p 2^et has passed 2^(R + 4)
                const int et = tops.y;
                const bool wide = tops.w != 0;
                const bool grow = mx > m + 4.0f || (m == -INFINITY && mx > m);
                float f = 1.0f;
                if (grow) {
                    const float d = m == -INFINITY ? -4096.0f : fmaxf(m - mx, -4096.0f), whole = floorf(d);
                    l *= t5_ex2(d);
                    f = m == -INFINITY ? 0.0f : t5_ex2(d - whole);
                    R = m == -INFINITY ? et - 4096 : R + (int)whole;
                    m = mx;
                }
                const float mref = m == -INFINITY ? 0.0f : -m;
                int top = et + (int)floorf(fminf(fmaxf(mx + mref, -4096.0f), 64.0f)); // the tile's largest p 2^et
                int far = top; // what has to lie above R + 4 for R to follow
                if (wide) {
                    float w = 0.0f;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            w = fmaxf(w, t5_ex2(fmaf(y[c][k].x, down, mref)) * vscale[st][c * 32 + 2 * k]);
                            w = fmaxf(w, t5_ex2(fmaf(y[c][k].y, down, mref)) * vscale[st][c * 32 + 2 * k + 1]);
                        }
                    // (R not so low that 2^lift below is no float: 2^-3 and 2^10 are held alike in two halves)
                    top = w > 0.0f ? et + max((__float_as_int(w) >> 23) - 127, kPcHead - 127) : R;
                    far = w > 0.0f ? max(top, et + kPcHead + 4 - 127) : R;
                }
                const bool raise = mx > -INFINITY && far > R + 4;
                if (raise) {
                    f *= R - top < -126 ? 0.0f : exp2_int(R - top);
                    R = top;
                }
                since *= f;
                if (j % kFold != 0 && __any_sync(0xffffffffu, grow || raise)) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float o[32];
                        uint32_t w[32];
                        tmem_ld32(trow + S::kO + c * 32, o);
                        tc_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(o[k] * f);
                        tmem_st32(trow + S::kO + c * 32, w);
                    }
                }
                // ---- weights in units of 2^(R - head), their sum, and their two planes over the scores
                const int lift = max(et - R + kPcHead, -4096); // p 2^et 2^-(R - head) = 2^(s - m + lift)
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                if (!__any_sync(0xffffffffu, wide || lift < -64)) {
                    const float ref = mref + (float)lift;
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        uint32_t ph[16], pl[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float2 w = __ffma2_rn(y[c][k], make_float2(down, down), make_float2(ref, ref));
                            w = make_float2(t5_ex2(w.x), t5_ex2(w.y));
                            sum[k & 1] = __fadd2_rn(sum[k & 1], w);
                            split_half2(w.x, w.y, ph[k], pl[k]);
                        }
                        tmem_st16(trow + c * 32, ph);
                        tmem_st16(trow + c * 32 + 16, pl);
                    }
                    l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) * exp2_int(-min(lift, 126)); // (past 126 it is less than 2^-112 either way)
                } else { // the sum is taken before V's scales
                    const float fw = exp2_low(min(lift, 127)), fx = exp2_int(min(max(lift - 127, 0), 127)); // (past 127 in a narrow tile alone)
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        uint32_t ph[16], pl[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float2 w = make_float2(t5_ex2(fmaf(y[c][k].x, down, mref)), t5_ex2(fmaf(y[c][k].y, down, mref)));
                            sum[k & 1] = __fadd2_rn(sum[k & 1], w);
                            const float a = wide ? vscale[st][c * 32 + 2 * k] : fx, e = wide ? vscale[st][c * 32 + 2 * k + 1] : fx;
                            split_half2(w.x * a * fw, w.y * e * fw, ph[k], pl[k]);
                        }
                        tmem_st16(trow + c * 32, ph);
                        tmem_st16(trow + c * 32 + 16, pl);
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bars.p_ready[T]);
                if (j + 1 < nst) wait(&bars.kv_full[st ^ 1], ((j + 1) >> 1) & 1, 0x55);
            }
            wait(&bars.o_full, 0, 0x52);
            if (lost) give_up(lost);
            if (__all_sync(0xffffffffu, lost == 0)) {
                tc_fence_after();
                // 2^(R - head) in two steps: it may lie below what one float holds
                const float inv = (l > 0.0f ? 1.0f / l : 0.0f) * (1.0f / (1 << kPcHead)), unit = R < -126 ? 0.0f : exp2_int(min(R, 127));
                float4 v[HD / 4];
#pragma unroll
                for (int k = 0; k < HD / 4; ++k) {
                    const float4 *at = place(k);
                    v[k] = nst > kFold && live ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                __syncwarp(); // every lane has read before anything is written
                // 32 columns at a time through 4 KB of the warp's own (k-th four values of lane l at slot l ^ k of piece k), so that
                // a store writes four whole lines
                uint8_t *hold = HD <= 64 ? reinterpret_cast<uint8_t *>(place(0) - lane) : smem + S::kOffSum + warp * 4096;
                constexpr int kPiece = HD <= 64 ? kPcRows * 16 : 512;
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    float o[32];
                    tmem_ld32(trow + S::kO + c * 32, o);
                    tc_wait_ld();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float4 w = v[8 * c + k];
                        *reinterpret_cast<float4 *>(hold + k * kPiece + (lane ^ k) * 16) =
                            l > 0.0f ? make_float4(fmaf(w.x, since, o[4 * k]) * inv * unit, fmaf(w.y, since, o[4 * k + 1]) * inv * unit,
                                                   fmaf(w.z, since, o[4 * k + 2]) * inv * unit, fmaf(w.w, since, o[4 * k + 3]) * inv * unit)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int row = 4 * k + (lane >> 3), q = lane & 7;
                        const float4 w = *reinterpret_cast<const float4 *>(hold + q * kPiece + (row ^ q) * 16);
                        float *to = reinterpret_cast<float *>(__shfl_sync(0xffffffffu, (uint64_t)dst, row));
                        if (__shfl_sync(0xffffffffu, (int)live, row)) *reinterpret_cast<float4 *>(to + c * 32 + q * 4) = w;
                    }
                    __syncwarp();
                }
                if (live && p.splits > 1) *reinterpret_cast<float2 *>(dst + HD) = make_float2(m, l);
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ================= converters: 64 bytes (HD 32: 32) of one key's K and V each =================
        constexpr int NP = HD == 32 ? 2 : 4; // pieces of 16 codes
        const int ct = tid - kPcSoft, key = ct % BN, piece0 = (ct / BN) * NP;
        auto look = [&](int j) -> int64_t { // row of this thread's key in the pool, -1: not there
            const int k = kb0 + j * BN + key;
            if (j >= nst || k < rr.lo || k >= rr.hi) return -1;
            const int pi = k / p.pv.page_size, page = p.pv.page(b, pi);
            if (page < 0) {
                p.pv.raise(FBLT_PAGED_BAD_PAGE);
                return -1;
            }
            return p.pv.row(page, kvh, k - pi * p.pv.page_size);
        };
        uint4 kr[NP], vr[NP];
        int ek = 0, ev = 0;
        bool here = false;
        auto load = [&](int64_t row) { // a key that is not there: zeros
            here = row >= 0;
            ek = ev = 0;
#pragma unroll
            for (int i = 0; i < NP; ++i) kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
            if (here) {
                const uint4 *kp = reinterpret_cast<const uint4 *>(p.pv.kc + row * HD) + piece0;
                const uint4 *vp = reinterpret_cast<const uint4 *>(p.pv.vc + row * HD) + piece0;
#pragma unroll
                for (int i = 0; i < NP; ++i) kr[i] = __ldg(kp + i);
#pragma unroll
                for (int i = 0; i < NP; ++i) vr[i] = __ldg(vp + i);
                ek = min(max((int)p.pv.ke[row], F::kEmin), F::kEmax);
                ev = min(max((int)p.pv.ve[row], F::kEmin), F::kEmax);
            }
        };
        // whether this thread's part of a row holds anything but zeros
        auto any_value = [&](const uint4(&raw)[NP]) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < NP; ++i) w |= raw[i].x | raw[i].y | raw[i].z | raw[i].w;
            return (FMT == FBLT_KV_E4M3 ? w & 0x7f7f7f7fu : w) != 0;
        };
        load(look(0));
        int64_t next = look(1);
        for (int j = 0; j < nst; ++j) {
            const int st = j & 1;
            const bool lost = j >= 2 && !mbar_wait_abort(&bars.kv_empty[st], ((j >> 1) - 1) & 1, abortp);
            if (lost && lane == 0) give_up(0x53);
            // ---- the tile's range of exponents (keys that are there)
            {
                // (a row of zeros has the least exponent: it does not make a tile wide)
                bool sk = here && ek > F::kEmin, sv = here && ev > F::kEmin;
                if (__any_sync(0xffffffffu, here && !(sk && sv))) {
                    sk = here && (sk || any_value(kr));
                    sv = here && (sv || any_value(vr));
                }
                const int4 r = make_int4(__reduce_max_sync(0xffffffffu, here ? ek : -1000), __reduce_min_sync(0xffffffffu, sk ? ek : 1000),
                                         __reduce_max_sync(0xffffffffu, here ? ev : -1000), __reduce_min_sync(0xffffffffu, sv ? ev : 1000));
                if (lane == 0) range[st][warp - 8] = r;
            }
            if (converters_or(lost)) break; // all four warps go on or none
            int4 e = range[st][0];
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                const int4 r = range[st][i];
                e = make_int4(max(e.x, r.x), min(e.y, r.y), max(e.z, r.z), min(e.w, r.w));
            }
            const bool none = e.x < F::kEmin, kwide = e.x - e.y > kPcNarrow, vwide = e.z - e.w > kPcNarrow;
            const int kbelow = here ? e.x - ek : 0, vbelow = here ? e.z - ev : 0; // 2^-below: into the halves or the columns
            if (ct == 0) *reinterpret_cast<int4 *>(top_of[st]) = make_int4(none ? 0 : e.x, none ? 0 : e.z - (vwide ? kVUp : 0), kwide, vwide);
            const uint32_t vote = __ballot_sync(0xffffffffu, here);
            if (piece0 == 0) {
                kunder[st][key] = kbelow;
                vscale[st][key] = exp2_int(kVUp - vbelow);
                if ((lane & 15) == 0) present[st][key / 16] = ((vote >> lane) & 0xffff) != 0;
            }
            auto put = [&](uint8_t *dst, const uint4(&raw)[NP], __half2 s) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                    uint32_t x[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        F::halves(w[k], x[2 * k], x[2 * k + 1]);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            __half2 &hv = *reinterpret_cast<__half2 *>(&x[2 * k + q]);
                            hv = __hmul2(hv, s); // exact: a code has 8 bits, and 2^-4 of the least is a half
                        }
                    }
                    *reinterpret_cast<uint4 *>(dst + (piece0 + i) * 2 * (BN * 16)) = make_uint4(x[0], x[1], x[2], x[3]);
                    *reinterpret_cast<uint4 *>(dst + ((piece0 + i) * 2 + 1) * (BN * 16)) = make_uint4(x[4], x[5], x[6], x[7]);
                }
            };
            uint8_t *kd = smem + S::kOffKv + st * 2 * S::kKv + key * 16;
            put(kd, kr, __float2half2_rn(kwide ? 1.0f : kbelow > 24 ? 0.0f : exp2_int(-kbelow)));
            put(kd + S::kKv, vr, __float2half2_rn(vwide ? 1.0f : vbelow > 24 ? 0.0f : exp2_int(-vbelow)));
            fence_async_smem();
            mbar_arrive(&bars.kv_full[st]);
            load(next);
            next = look(j + 2);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 12) {
            // ================= issuer (the warp goes along, one lane issues) =================
            constexpr uint32_t kIdS = pc_idesc(BN, false), kIdO = pc_idesc(HD, true);
            // S = Q K^T: a 16-deep product reads two 8-column core matrices, BN (128) rows apart
            auto issue_s = [&](int T, int st) {
                const uint32_t q = tmem + S::kQ + T * S::kQTile, k = sbase + S::kOffKv + st * 2 * S::kKv, d = tmem + T * S::kTile;
                if (elect_one()) {
#pragma unroll
                    for (int pl = 1; pl >= 0; --pl)
#pragma unroll
                        for (int s = 0; s < HD / 16; ++s) {
                            const uint64_t kd = t5_desc(k + s * 2 * (BN * 16), BN * 16, 128);
                            if (HD == 128 && pl == 1)
                                mma_f16_ss(d, t5_desc(sbase + T * S::kQPlane + s * 2 * (kPcRows * 16), kPcRows * 16, 128), kd, kIdS, s > 0);
                            else
                                mma_f16_ts(d, q + pl * S::kQCols + s * 8, kd, kIdS, pl == 0 || s > 0);
                        }
                    tc_commit(&bars.s_full[T]);
                }
                __syncwarp();
            };
            bool ok = warp_wait(&bars.q_full, 0, abortp);
            if (ok) {
                ok = warp_wait(&bars.kv_full[0], 0, abortp);
                if (ok) {
                    tc_fence_after();
                    for (int T = 0; T < tiles; ++T) issue_s(T, 0);
                }
                for (int j = 0; j < nst && ok; ++j) {
                    const int st = j & 1;
                    for (int T = 0; T < tiles; ++T) {
                        ok = warp_wait(&bars.p_ready[T], j & 1, abortp);
                        if (!ok) break;
                        tc_fence_after();
                        // O += P V: 16 keys are two 8-row core matrices of V, 128 bytes apart; 8 columns of O the next BN rows on
                        const uint32_t v = sbase + S::kOffKv + st * 2 * S::kKv + S::kKv, a = tmem + T * S::kTile, d = a + S::kO;
                        if (elect_one()) {
#pragma unroll
                            for (int pl = 1; pl >= 0; --pl)
#pragma unroll
                                for (int s = 0; s < BN / 16; ++s)
                                    mma_f16_ts(d, a + (s >> 1) * 32 + pl * 16 + (s & 1) * 8, t5_desc(v + s * 256, 128, BN * 16), kIdO,
                                               j % kFold != 0 || pl < 1 || s > 0);
                            if (T == tiles - 1) tc_commit(&bars.kv_empty[st]);
                            if (j == nst - 1 && T == tiles - 1) tc_commit(&bars.o_full);
                        }
                        __syncwarp();
                        if (j + 1 < nst) {
                            if (T == 0) {
                                ok = warp_wait(&bars.kv_full[st ^ 1], ((j + 1) >> 1) & 1, abortp);
                                if (!ok) break;
                                tc_fence_after();
                            }
                            issue_s(T, st ^ 1);
                        }
                    }
                }
            }
            if (!ok && lane == 0) give_up(0x54);
            // whatever was issued has completed before the TMEM is given back
            if (elect_one()) tc_commit(&bars.fin);
            __syncwarp();
            mbar_wait(&bars.fin, 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int HD, int FMT>
static int launch_chunk_t(const PagedAttnParams &p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (const int st = allow_smem((const void *)paged_chunk_kernel<HD, FMT>, PcShape<HD>::kSmem, done)) return st;
    paged_chunk_kernel<HD, FMT><<<paged_grid(p), kPcThreads, PcShape<HD>::kSmem, s>>>(p);
    count_launch();
    return check_launch("paged_chunk_kernel");
}

int launch_paged_chunk(const PagedAttnParams &p, int hd, bool e4, cudaStream_t s) {
    switch (hd) {
    case 32: return e4 ? launch_chunk_t<32, FBLT_KV_E4M3>(p, s) : launch_chunk_t<32, FBLT_KV_INT8>(p, s);
    case 64: return e4 ? launch_chunk_t<64, FBLT_KV_E4M3>(p, s) : launch_chunk_t<64, FBLT_KV_INT8>(p, s);
    default: return e4 ? launch_chunk_t<128, FBLT_KV_E4M3>(p, s) : launch_chunk_t<128, FBLT_KV_INT8>(p, s);
    }
}

int chunk_take_error() {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_chunk_error, sizeof(v)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_chunk_error, &zero, sizeof(zero));
    return (int)v;
}

} // namespace fblt
