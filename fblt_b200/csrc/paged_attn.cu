// Attention of new query rows over the 8-bit paged KV cache (fblt_paged_attn): the streaming kernel for few rows per
// (sequence, kv head) -- one token, a drafted block, with grouped heads up to 32 rows -- the merge of a split key
// range, and the dispatch.
//
// out = sum_k p_k v_k / sum_k p_k, p_k = 2^(s_k - m), s_k = scale log2(e) q . k, in one pass over the keys with the
// running maximum m. A cache row is used by at most G * n_new query rows, so the bytes of the cache bound this: the
// stream has to be read at HBM speed and everything else has to fit beside it.
//
//   * CTA = (sequence, kv head, key range); the rows of one kv head are its G query heads of every
//     new token, so grouped heads and drafted blocks read a key once.
//   * Stages of 64 keys (head_dim 128: 32), four groups that lie in one page each, are copied ahead into shared memory:
//     by every warp for itself, or, where warps share the keys, by a producer warp; group i lies 32 bytes further round
//     the banks than group i - 1.
//   * Four consumer warps multiply with mma.sync m16n8k16 in fp16: codes ARE halves (an 8-bit code has at most 8
//     significant bits), and the 16 rows of the A operand are 8 query rows in two planes, q = hi + lo with 22 bits
//     in all, so q . code is fp32 class in ONE instruction and hi + lo are added in registers. Probabilities go back
//     the same way for P V. The exponents of K multiply scores, those of V probabilities: per (row, key), not per value.
//     tcgen05 would need 128 rows of A; 8 .. 32 exist.
//   * Both products see keys and head_dim in an order of our own choosing (a sum has none): lane t of a quad takes 16
//     neighbouring codes of a K row, lane g 1/8 of a V row, and the 16 keys of one product are 4 of each group, so
//     that with the 32-byte skew V's column-wise reads touch every bank once.
//
// Measured (B200): one token of 256 sequences of up to 4 k keys, 16 kv heads, head_dim 64, int8: 273-284 us, 4.0 TB/s of
// the cache's bytes; 8 rows x 4 heads over 64 caches of up to 8 k keys, head_dim 128, e4m3: 403-408 us. HBM's bound would
// be 171 and 102 us: what is left is the conversion of codes to halves (five instructions for four int8 codes) and its
// latency with 12 warps on an SM, which registers limit: issue slots are half busy, and warps that share keys each convert
// all of them. Measured and slower: a producer warp where warps share nothing 332 us; stages of 32 keys at head_dim 64
// 531 us; a warp's 8 rows in steps of 16 keys instead of 32 456 us; four CTAs an SM at head_dim 128 519 us; a maximum that
// moves with every larger score (not by 2^4 at least) 8 us more.
#include "paged.cuh"

namespace fblt {

__device__ unsigned int g_paged_error; // 0 = ok; otherwise (code << 24) | blockIdx.x of the first CTA that gave up

// A row's weights times the scales of V, p 2^ev, are put into halves in units of 2^(R - kPsHead), R within four of the
// largest exponent that p 2^ev has had (R follows the row's maximum when that moves): at most 2^(kPsHead + 5), and what
// is 2^-24 of the largest still has 11 bits, however unequal the rows of V are.
// The tensor cores cut every sum off below 24 bits, a pull towards zero of about 2e-8 a product (5e-6 over 4800 keys):
// after so many keys what they hold is added, rounded, to sums of its own.
constexpr int kPsFold = 256;
constexpr int kPsHead = 10, kPsNoUnit = -(1 << 20);
constexpr float kPsLazy = 4.0f; // a row's m moves, and what it holds is rescaled, once a score lies 2^4 above it

template <int HD>
struct PsShape {
    static constexpr int kKeys = HD == 128 ? 32 : 64;   // keys of a stage
    static constexpr int kPer = kKeys / 4;              // keys of a group
    static constexpr int kGroup = kPer * HD;            // their bytes
    static constexpr int kPitch = kGroup + 32;          // see the bank skew above
    static constexpr int kOffV = 4 * kPitch, kOffE = 8 * kPitch;
    static constexpr int kStage = 8 * kPitch + 128; // K groups, V groups, exponents
};

template <int HD, int RB, int WR>
struct PsCta {
    // Where 64 tensor core accumulators a thread and 32 folded sums would leave room for few warps, the sums, touched every
    // 256 keys, live in shared memory (8 rows x 4 heads, head_dim 128: two CTAs with sums in registers 526 us, three with
    // shared ones 516 us, and with the pieces below 459 and 429 us; 6 rows x 4 heads, head_dim 64: 327 and 266 us).
    static constexpr bool kSharedSum = RB * HD >= 128 && WR > 1;
    static constexpr int kMin = !kSharedSum ? 1 : HD == 128 ? 3 : 2;        // CTAs of an SM
    static constexpr int kStages = kSharedSum && HD == 128 ? 4 : 8; // of the CTA; a warp's own: a quarter
    static constexpr int kBytes = kStages * PsShape<HD>::kStage + RB * WR * (HD / 16) * 512 + (kSharedSum ? RB * (HD / 8) * 1024 : 0);
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// 16 bytes global -> shared, bypassing L1
__device__ __forceinline__ void cp_async_16(void *smem_dst, const void *gmem_src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}
__device__ __forceinline__ void cp_async_8(void *smem_dst, const void *gmem_src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int HD, int FMT, int RB, int WR>
__global__ void __launch_bounds__(WR == 1 ? 128 : 160, PsCta<HD, RB, WR>::kMin) paged_stream_kernel(const PagedAttnParams p) {
    using F = KvFormat<FMT>;
    using S = PsShape<HD>;
    constexpr int WK = 4 / WR, RT = 8 * RB * WR, KS = HD / 16, NB = HD / 8, PR = HD + 4, NS = PsCta<HD, RB, WR>::kStages;
    constexpr bool SS = PsCta<HD, RB, WR>::kSharedSum;
    constexpr int U = RB * HD >= 256 ? 1 : 2; // products of 16 keys that go through the softmax together
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    uint4 *sq = reinterpret_cast<uint4 *>(smem + NS * S::kStage); // [RB * WR][KS][32] A fragments
    __shared__ uint64_t full[NS], empty[NS]; // WR > 1
    __shared__ uint32_t vmask[NS];
    __shared__ float crow[RT], sm[WK * RT], sl[WK * RT];
    __shared__ __align__(16) float scale[4][2][S::kKeys]; // a warp's own: the stage's scales of K and of V
    __shared__ int s_abort;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedCtaAt at = paged_cta(p);
    const int kvh = at.kvh, split = at.split, b = at.unit; // one tile of rows: the plan's RT holds them all
    int r0, n, base;
    if (!paged_seq(p.pv, p.cu, p.base, p.total, b, r0, n, base)) return;
    if (n > p.max_new) {
        if (tid == 0) p.pv.raise(FBLT_PAGED_BAD_LENGTH);
    }
    const int rows = min(n, p.max_new) * p.G;
    if (rows == 0) return;
    const RowRange rr = tile_range(p, base, n, 0, rows);
    // this split's stages (a stage starts at a multiple of 16, a page too)
    const int first = rr.lo & ~15, stages = (rr.hi - first + S::kKeys - 1) / S::kKeys, per = (stages + p.splits - 1) / p.splits;
    const int st0 = min(stages, split * per), nst = min(stages, st0 + per) - st0;
    const int kb0 = first + st0 * S::kKeys;

    if (WR > 1 && tid == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], 33);
            mbar_init(&empty[i], WR);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // Rows of the pool where this lane's group begins, -1: not there. Eight stages at a time, a lane per group: stage
    // first + every * (lane / 4), group lane % 4.
    auto look = [&](int first, int every) -> int64_t {
        const int st = first + every * (lane >> 2), key = kb0 + st * S::kKeys + (lane & 3) * S::kPer;
        if (st >= nst || key >= rr.hi) return -1;
        const int pi = key / p.pv.page_size, page = p.pv.page(b, pi);
        if (page < 0) p.pv.raise(FBLT_PAGED_BAD_PAGE);
        return page < 0 ? -1 : p.pv.row(page, kvh, key - pi * p.pv.page_size);
    };

    if (WR > 1 && warp == 4) {
        // ---- producer; pages are looked up eight stages ahead
        int64_t now = -1, next = look(0, 1);
        for (int st = 0; st < nst; ++st) {
            const int slot = st % NS;
            if ((st & 7) == 0) {
                now = next;
                next = look(st + 8, 1);
            }
            const int64_t at = __shfl_sync(0xffffffffu, now, (st & 7) * 4 + (lane & 3));
            const uint32_t ok = __ballot_sync(0xffffffffu, at >= 0) & 15;
            if (st >= NS) {
                bool good = true;
                if (lane == 0) good = mbar_wait_abort(&empty[slot], ((st / NS) - 1) & 1, (const volatile int *)&s_abort);
                if (!__shfl_sync(0xffffffffu, good, 0)) {
                    if (lane == 0) {
                        *(volatile int *)&s_abort = 1;
                        atomicCAS(&g_paged_error, 0u, (0x41u << 24) | (blockIdx.x & 0xffffffu));
                    }
                    break;
                }
            }
            uint8_t *stage = ring + slot * S::kStage;
            if (lane == 0) {
                vmask[slot] = ok;
                mbar_expect_tx(&full[slot], __popc(ok) * 2 * S::kGroup);
            }
            __syncwarp();
            // lane = (group, K / V): its codes as one bulk copy, its exponents in eights
            const int64_t row = __shfl_sync(0xffffffffu, at, (lane >> 1) & 3);
            if (lane < 8 && row >= 0) {
                const int gi = lane >> 1, v = lane & 1;
                bulk_load(stage + v * S::kOffV + gi * S::kPitch, (v ? p.pv.vc : p.pv.kc) + row * HD, S::kGroup, &full[slot]);
#pragma unroll
                for (int k = 0; k < S::kPer; k += 8)
                    cp_async_8(stage + S::kOffE + v * S::kKeys + gi * S::kPer + k, (v ? p.pv.ve : p.pv.ke) + row + k);
            }
            cp_async_arrive(&full[slot]); // one arrival a lane, when its exponents have landed
        }
        asm volatile("cp.async.wait_all;" ::: "memory"); // nothing is in flight when the CTA goes
    } else {
        // ---- consumers
        const int g = lane >> 2, t = lane & 3, wr = warp / WK, wk = warp % WK;
        // query fragments: a warp per block of 8 rows; row g's values at this lane's head_dim positions
        for (int rb = warp; rb < RB * WR; rb += 4) {
            const int r = rb * 8 + g;
            float4 x[KS];
            float a = 0.0f, odd = 0.0f; // odd: NaN once a value is not finite
            const bool live = r < rows;
            const int i = live ? r / p.G : 0;
            const float *src = p.q + (int64_t)(r0 + i) * p.qs + (int64_t)(kvh * p.G + (r - i * p.G)) * HD;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = HD == 32 ? 8 * t + 4 * s : 64 * (s >> 2) + 16 * t + 4 * (s & 3);
                x[s] = live ? *reinterpret_cast<const float4 *>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float v[4] = {x[s].x, x[s].y, x[s].z, x[s].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a = finite_f(v[e]) ? fmaxf(a, fabsf(v[e])) : a;
                    odd = fmaf(v[e], 0.0f, odd);
                }
            }
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
            odd += __shfl_xor_sync(0xffffffffu, odd, 1);
            odd += __shfl_xor_sync(0xffffffffu, odd, 2);
            // q * 2^e with its largest value in [2^13, 2^14): halves keep the row's small values too
            const int e = min(13 - ((__float_as_int(a) >> 23) - 127), 126);
            const float up = exp2_int(e);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint4 f;
                split_half2(x[s].x * up, x[s].y * up, f.x, f.y);
                split_half2(x[s].z * up, x[s].w * up, f.z, f.w);
                sq[(rb * KS + s) * 32 + lane] = f;
            }
            if (t == 0) crow[rb * 8 + g] = p.qscale * exp2_int(-e) + odd; // (NaN for a row that is not finite)
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");

        float m[RB], l[RB], c[RB];
        float o[RB][NB][4]; // the tensor cores' sums, a plane in each half
        // columns 2t and 2t + 1 of every block: what was folded
        float2 *ssum = reinterpret_cast<float2 *>(sq + RB * WR * KS * 32) + tid;
        float2 rsum[RB][SS ? 1 : NB];
        const auto sum = [&](int rb, int j) -> float2 & {
            if constexpr (SS) return ssum[(rb * NB + j) * 128];
            else return rsum[rb][j];
        };
        int lo[RB], span[RB], R[RB]; // o holds sums of p v in units of 2^R
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            // a row past the last one has zeros for a query and sees what the last one sees; it is not written
            const int ri = (wr * RB + rb) * 8 + g, pos = base + min(ri, rows - 1) / p.G;
            const int hi = p.block_mode ? base + n : pos + 1;
            lo[rb] = p.block_mode || p.window <= 0 ? 0 : max(0, pos - p.window + 1);
            span[rb] = hi - lo[rb];
            m[rb] = -INFINITY;
            l[rb] = 0.0f;
            R[rb] = kPsNoUnit;
            c[rb] = crow[ri];
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                o[rb][j][0] = o[rb][j][1] = o[rb][j][2] = o[rb][j][3] = 0.0f;
                sum(rb, j) = make_float2(0.0f, 0.0f);
            }
        }
        int held = 0; // stages in o
        auto fold = [&]() {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    sum(rb, j) = __fadd2_rn(sum(rb, j), __fadd2_rn(make_float2(o[rb][j][0], o[rb][j][1]), make_float2(o[rb][j][2], o[rb][j][3])));
                    o[rb][j][0] = o[rb][j][1] = o[rb][j][2] = o[rb][j][3] = 0.0f;
                }
            held = 0;
        };
        const uint4 *myq = sq + wr * RB * KS * 32 + lane;
        float(&kscale)[S::kKeys] = scale[warp][0], (&vscale)[S::kKeys] = scale[warp][1];
        // one stage: keys kb .., groups `here` of it have landed
        auto work = [&](uint8_t *stage, int kb, uint32_t here) {
            const bool there = (here >> t) & 1; // this lane's scores and V rows are keys of group t
            // every key of the stage is there and every row of the warp sees it
            const bool whole = __all_sync(0xffffffffu, here == 15 && kb >= lo[0] && kb + S::kKeys <= lo[0] + span[0] &&
                                                           (RB == 1 || (kb >= lo[RB - 1] && kb + S::kKeys <= lo[RB - 1] + span[RB - 1])));
            // Slots that hold no visible key may hold any bytes, NaN codes too, and zero times those is no zero: their V
            // rows are cleared (every warp of the share clears them before it reads, so no one sees them).
            if (here != 15 || kb < rr.lo || kb + S::kKeys > rr.hi) {
                for (int i = lane; i < S::kKeys * (HD / 16); i += 32) {
                    const int k = i / (HD / 16), grp = k / S::kPer;
                    if (kb + k < rr.lo || kb + k >= rr.hi || !((here >> grp) & 1))
                        *reinterpret_cast<uint4 *>(stage + S::kOffV + grp * S::kPitch + (k % S::kPer) * HD + (i % (HD / 16)) * 16) =
                            make_uint4(0, 0, 0, 0);
                }
                // the producer's next bulk copy into this stage goes through the async proxy: it comes behind these stores
                if (WR > 1) fence_async_smem();
            }
            // ---- scales of the stage's keys; V's in units of 2^et, kVUp below the largest
            int et = kPsNoUnit;
            {
                constexpr int KL = S::kKeys / 32; // keys of a lane
                int e[KL];
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int k = lane * KL + i;
                    kscale[k] = exp2_int(min(max((int)(int8_t)stage[S::kOffE + k], F::kEmin), F::kEmax));
                    e[i] = min(max((int)(int8_t)stage[S::kOffE + S::kKeys + k], F::kEmin), F::kEmax);
                    if (kb + k >= rr.lo && kb + k < rr.hi && ((here >> (k / S::kPer)) & 1)) et = max(et, e[i]);
                }
                et = __reduce_max_sync(0xffffffffu, et);
#pragma unroll
                for (int i = 0; i < KL; ++i) vscale[lane * KL + i] = exp2_int(min(max(e[i] - et, -kVSpan), 0) + kVUp);
                et -= kVUp;
            }
            __syncwarp();
#pragma unroll 1
            for (int u0 = 0; u0 < S::kPer / 4; u0 += U) {
                // ---- S: K rows of this lane are keys 4u + (g & 1) and 4u + (g & 1) + 2 of group g / 2
                float s[RB][U][2][4];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) s[rb][u][nb][0] = s[rb][u][nb][1] = s[rb][u][nb][2] = s[rb][u][nb][3] = 0.0f;
                const uint8_t *krow = stage + (g >> 1) * S::kPitch + (4 * u0 + (g & 1)) * HD;
#pragma unroll
                for (int i = 0; i < (HD + 63) / 64; ++i) {
                    constexpr int KW = HD == 32 ? 2 : 4;
                    uint32_t kw[U][2][KW];
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) {
                            const uint8_t *src = krow + (4 * u + 2 * nb) * HD;
                            if (HD == 32) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(src + 8 * t);
                                kw[u][nb][0] = v.x, kw[u][nb][1] = v.y;
                            } else {
                                const uint4 v = *reinterpret_cast<const uint4 *>(src + 64 * i + 16 * t);
                                kw[u][nb][0] = v.x, kw[u][nb][1] = v.y, kw[u][nb][KW - 2] = v.z, kw[u][nb][KW - 1] = v.w;
                            }
                        }
#pragma unroll
                    for (int w = 0; w < KW; ++w) {
                        uint4 a[RB];
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) a[rb] = myq[(rb * KS + 4 * i + w) * 32];
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int nb = 0; nb < 2; ++nb) {
                                uint32_t b0, b1;
                                F::halves(kw[u][nb][w], b0, b1);
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) mma_f16(s[rb][u][nb], a[rb], b0, b1);
                            }
                    }
                }
                // ---- softmax: this lane has row g of every block and keys 4u .. 4u + 3 of group t
                const int kl = t * S::kPer + 4 * u0; // key within the stage
                float2 x[RB][U][2];
                float mn[RB], odd = 0.0f; // odd: NaN once a score is not finite
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) mn[rb] = -INFINITY;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float4 ks = *reinterpret_cast<const float4 *>(&kscale[kl + 4 * u]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) {
                            const float(&v)[4] = s[rb][u][nb];
                            float2 y = __fadd2_rn(make_float2(v[0], v[1]), make_float2(v[2], v[3]));
                            // both powers of two first: one of them may be what keeps the other's product in fp32's range
                            y = __fmul2_rn(y, __fmul2_rn(nb ? make_float2(ks.z, ks.w) : make_float2(ks.x, ks.y), make_float2(c[rb], c[rb])));
                            x[rb][u][nb] = y;
                            odd = fmaf(y.x, 0.0f, fmaf(y.y, 0.0f, odd));
                            mn[rb] = fmaxf(mn[rb], fmaxf(y.x, y.y));
                        }
                }
                if (!whole || __any_sync(0xffffffffu, odd != 0.0f)) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        mn[rb] = -INFINITY;
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int nb = 0; nb < 2; ++nb) {
                                float2 &y = x[rb][u][nb];
                                const int k = kb + kl + 4 * u + 2 * nb - lo[rb];
                                // a product of 0 times a scale past fp32's range
                                if (isnan(y.x) && !isnan(c[rb])) y.x = 0.0f;
                                if (isnan(y.y) && !isnan(c[rb])) y.y = 0.0f;
                                y.x = there && (unsigned)k < (unsigned)span[rb] && finite_f(y.x) ? y.x : -INFINITY;
                                y.y = there && (unsigned)(k + 1) < (unsigned)span[rb] && finite_f(y.y) ? y.y : -INFINITY;
                                mn[rb] = fmaxf(mn[rb], fmaxf(y.x, y.y));
                            }
                    }
                }
                bool moved = false;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    mn[rb] = fmaxf(mn[rb], __shfl_xor_sync(0xffffffffu, mn[rb], 1));
                    mn[rb] = fmaxf(mn[rb], __shfl_xor_sync(0xffffffffu, mn[rb], 2));
                    mn[rb] = fmaxf(mn[rb], m[rb]);
                    moved |= mn[rb] > m[rb] + kPsLazy;
                    mn[rb] = mn[rb] > m[rb] + kPsLazy ? mn[rb] : m[rb];
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        // o's unit follows the maximum down, so its values shrink by less than 2
                        const float d = m[rb] == -INFINITY ? 0.0f : fmaxf(m[rb] - mn[rb], -4096.0f), down = floorf(d);
                        const float f = t5_ex2(d - down);
                        l[rb] *= t5_ex2(d);
                        R[rb] += (int)down;
                        m[rb] = mn[rb];
#pragma unroll
                        for (int j = 0; j < NB; ++j) {
                            o[rb][j][0] *= f, o[rb][j][1] *= f, o[rb][j][2] *= f, o[rb][j][3] *= f;
                            sum(rb, j) = __fmul2_rn(sum(rb, j), make_float2(f, f));
                        }
                    }
                }
                float top[RB]; // the largest p 2^(ev - et)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float mref = m[rb] == -INFINITY ? 0.0f : -m[rb];
                    float2 add = make_float2(0.0f, 0.0f);
                    top[rb] = 0.0f;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const float4 vs = *reinterpret_cast<const float4 *>(&vscale[kl + 4 * u]);
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) {
                            float2 &y = x[rb][u][nb];
                            y = __fadd2_rn(y, make_float2(mref, mref));
                            y = make_float2(t5_ex2(y.x), t5_ex2(y.y));
                            add = __fadd2_rn(add, y);
                            y = __fmul2_rn(y, nb ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y));
                            top[rb] = fmaxf(top[rb], fmaxf(y.x, y.y));
                        }
                    }
                    l[rb] += add.x + add.y;
                }
                bool raise = false;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) // (or where R lies below its least, see there)
                    raise |= top[rb] > 0.0f && max(__float_as_int(top[rb]) >> 23, kPsHead + 4) > R[rb] + 4 + 127 - et;
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        float w = fmaxf(top[rb], __shfl_xor_sync(0xffffffffu, top[rb], 1));
                        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
                        // (R not so low that 2^(et - R + kPsHead) below is no float: 2^-3 and 2^10 are held alike in two halves)
                        const int Rn = w > 0.0f ? max(R[rb], et + max((__float_as_int(w) >> 23) - 127, kPsHead - 127)) : R[rb];
                        const float f = R[rb] - Rn < -126 ? 0.0f : exp2_int(R[rb] - Rn);
                        R[rb] = Rn;
#pragma unroll
                        for (int j = 0; j < NB; ++j) {
                            o[rb][j][0] *= f, o[rb][j][1] *= f, o[rb][j][2] *= f, o[rb][j][3] *= f;
                            sum(rb, j) = __fmul2_rn(sum(rb, j), make_float2(f, f));
                        }
                    }
                }
                uint4 pa[RB][U];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    // p 2^(ev - et) in units of 2^(R - kPsHead); a row without a weight has only zeros
                    const float f = exp2_low(min(et - R[rb] + kPsHead, 127));
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        split_half2(x[rb][u][0].x * f, x[rb][u][0].y * f, pa[rb][u].x, pa[rb][u].y);
                        split_half2(x[rb][u][1].x * f, x[rb][u][1].y * f, pa[rb][u].z, pa[rb][u].w);
                    }
                }
                // ---- O += P V: columns g * HD / 8 .. of keys 4u .. 4u + 3 of group t
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint8_t *vrow = stage + S::kOffV + t * S::kPitch + 4 * (u0 + u) * HD + g * NB;
                    uint32_t vw[4][NB / 4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (HD == 32) {
                            vw[j][0] = *reinterpret_cast<const uint32_t *>(vrow + j * HD);
                        } else if (HD == 64) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(vrow + j * HD);
                            vw[j][0] = v.x, vw[j][NB / 4 - 1] = v.y;
                        } else {
                            const uint4 v = *reinterpret_cast<const uint4 *>(vrow + j * HD);
                            vw[j][0] = v.x, vw[j][1 % (NB / 4)] = v.y, vw[j][2 % (NB / 4)] = v.z, vw[j][3 % (NB / 4)] = v.w;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < NB / 4; ++w) {
                        uint32_t b0[4], b1[4];
                        F::halves(__byte_perm(vw[0][w], vw[1][w], 0x5140), b0[0], b0[1]);
                        F::halves(__byte_perm(vw[0][w], vw[1][w], 0x7362), b0[2], b0[3]);
                        F::halves(__byte_perm(vw[2][w], vw[3][w], 0x5140), b1[0], b1[1]);
                        F::halves(__byte_perm(vw[2][w], vw[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb) mma_f16(o[rb][4 * w + j], pa[rb][u], b0[j], b1[j]);
                    }
                }
            }
            if (++held == kPsFold / S::kKeys) fold();
        };
        if constexpr (WR == 1) {
            // The warp copies its own stages (wk, wk + 4, ..): sixteen bytes a lane and copy, two stages in turn. One producer
            // for all four warps spent 1450 clocks a stage on issuing them, half of what a warp spends on using one.
            uint8_t *mine = ring + warp * (NS / 4) * S::kStage;
            const int count = (nst - wk + 3) / 4;
            int64_t now = -1, next = look(wk, 4);
            uint32_t flying = 0; // groups of stage i at bits 4 (i % 2) ..
            auto fetch = [&](int i) { // i ascends by one
                if ((i & 7) == 0) {
                    now = next;
                    next = look(wk + 4 * (i + 8), 4);
                }
                const int64_t at = __shfl_sync(0xffffffffu, now, (i & 7) * 4 + (lane & 3));
                const uint32_t ok = i < count ? __ballot_sync(0xffffffffu, at >= 0) & 15 : 0;
                flying = (flying & ~(15u << 4 * (i & 1))) | ok << 4 * (i & 1);
                uint8_t *stage = mine + (i & 1) * S::kStage;
#pragma unroll
                for (int gi = 0; gi < 4; ++gi) {
                    const int64_t row = __shfl_sync(0xffffffffu, at, gi);
                    if (!((ok >> gi) & 1)) continue;
                    const uint8_t *ksrc = p.pv.kc + row * HD + lane * 16, *vsrc = p.pv.vc + row * HD + lane * 16;
                    uint8_t *kdst = stage + gi * S::kPitch + lane * 16;
#pragma unroll
                    for (int c = 0; c < S::kGroup; c += 512) {
                        cp_async_16(kdst + c, ksrc + c);
                        cp_async_16(kdst + S::kOffV + c, vsrc + c);
                    }
                    if (lane < S::kPer / 4) // K's exponents, then V's, eight at a time
                        cp_async_8(stage + S::kOffE + (lane & 1) * S::kKeys + gi * S::kPer + (lane >> 1) * 8,
                                   ((lane & 1) ? p.pv.ve : p.pv.ke) + row + (lane >> 1) * 8);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            static_assert(NS / 4 == 2, "two stages a warp");
            fetch(0);
            fetch(1);
            for (int i = 0; i < count; ++i) {
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp();
                work(mine + (i & 1) * S::kStage, kb0 + (wk + 4 * i) * S::kKeys, (flying >> 4 * (i & 1)) & 15);
                __syncwarp();
                fetch(i + 2);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            for (int st = wk; st < nst; st += WK) { // a stage belongs to the WR warps of one key share
                const int slot = st % NS;
                if (!warp_wait(&full[slot], (st / NS) & 1, (const volatile int *)&s_abort)) {
                    *(volatile int *)&s_abort = 1;
                    if (lane == 0) atomicCAS(&g_paged_error, 0u, (0x42u << 24) | (blockIdx.x & 0xffffffu));
                    break;
                }
                work(ring + slot * S::kStage, kb0 + st * S::kKeys, vmask[slot]);
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[slot]);
            }
        }
        fold();
        // ---- the warps' shares of the keys meet in shared memory (every copy has landed: the ring is free)
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float *part = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = wk * RT + (wr * RB + rb) * 8 + g;
            const float unit = R[rb] < -126 ? 0.0f : exp2_int(R[rb]);
            l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 1);
            l[rb] += __shfl_xor_sync(0xffffffffu, l[rb], 2);
            if (t == 0) {
                sm[row] = m[rb];
                sl[row] = l[rb];
            }
            constexpr float kDown = 1.0f / (float)(1 << kPsHead);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NB; j += 4) {
                    float4 v;
                    v.x = (h ? sum(rb, j).y : sum(rb, j).x) * kDown * unit;
                    v.y = (h ? sum(rb, j + 1).y : sum(rb, j + 1).x) * kDown * unit;
                    v.z = (h ? sum(rb, j + 2).y : sum(rb, j + 2).x) * kDown * unit;
                    v.w = (h ? sum(rb, j + 3).y : sum(rb, j + 3).x) * kDown * unit;
                    *reinterpret_cast<float4 *>(part + row * PR + (2 * t + h) * NB + j) = v;
                }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (WR > 1 && *(volatile int *)&s_abort) return;
        for (int it = tid; it < RT * (HD / 4); it += 128) {
            const int ri = it / (HD / 4), d = (it - ri * (HD / 4)) * 4, r = ri;
            if (r >= rows) continue;
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; ++k) M = fmaxf(M, sm[k * RT + ri]);
            const float mref = M == -INFINITY ? 0.0f : M;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.0f;
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float f = t5_ex2(sm[k * RT + ri] - mref);
                const float4 v = *reinterpret_cast<const float4 *>(part + (k * RT + ri) * PR + d);
                L += sl[k * RT + ri] * f;
                a.x += v.x * f, a.y += v.y * f, a.z += v.z * f, a.w += v.w * f;
            }
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
            a = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            const int i = r / p.G, head = kvh * p.G + (r - i * p.G);
            if (p.splits > 1) {
                float *w = p.ws + (((int64_t)(r0 + i) * p.H + head) * p.splits + split) * PR;
                *reinterpret_cast<float4 *>(w + d) = a;
                if (d == 0) *reinterpret_cast<float2 *>(w + HD) = make_float2(M, L);
            } else {
                *reinterpret_cast<float4 *>(p.out + (int64_t)(r0 + i) * p.os + (int64_t)head * HD + d) = a;
            }
        }
    }
}

// Merge of a split key range: HD / 4 lanes per (packed row, head), o = sum_s L_s 2^(m_s - M) o_s / sum_s L_s 2^(m_s - M).
// Every piece of a live row was written by the launch before, an empty one with L = 0.
template <int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnParams p) {
    constexpr int LPH = HD / 4, PR = HD + 4;
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPH;
    const int lane = threadIdx.x % LPH;
    if (unit >= (int64_t)p.total * p.H) return;
    const int r = (int)(unit / p.H), head = (int)(unit - (int64_t)r * p.H);
    int lo = 0, hi = p.batch; // the last sequence that starts at or before r
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid) <= r) lo = mid;
        else hi = mid;
    }
    int r0, n, base;
    if (!paged_seq(p.pv, p.cu, p.base, p.total, lo, r0, n, base) || r < r0 || r >= r0 + min(n, p.max_new)) return;
    const float *w = p.ws + unit * p.splits * PR;
    float M = -INFINITY, L = 0.0f;
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, w[s * PR + HD]);
    const float mref = M == -INFINITY ? 0.0f : M;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
        const float2 ml = *reinterpret_cast<const float2 *>(w + s * PR + HD);
        const float f = t5_ex2(ml.x - mref) * ml.y;
        const float4 v = *reinterpret_cast<const float4 *>(w + s * PR + lane * 4);
        L += f;
        a.x += v.x * f, a.y += v.y * f, a.z += v.z * f, a.w += v.w * f;
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    *reinterpret_cast<float4 *>(p.out + (int64_t)r * p.os + (int64_t)head * HD + lane * 4) =
        make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
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
    if ((int64_t)d->max_new * (d->num_heads / d->cache.num_kv_heads) > INT_MAX / 2)
        return fail(FBLT_ERR_LIMIT, "%s: max_new * num_heads / num_kv_heads exceeds 2^30", who);
    if (d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return FBLT_OK;
    if (!d->cu_new || !d->base_len || !d->q || !d->out) return fail(FBLT_ERR_ARG, "%s: NULL buffer", who);
    const int64_t E = (int64_t)d->num_heads * d->cache.head_dim;
    if (d->q_stride < E || d->out_stride < E) return fail(FBLT_ERR_ARG, "%s: row stride smaller than num_heads*head_dim", who);
    if ((d->q_stride | d->out_stride) & 3) return fail(FBLT_ERR_ARG, "%s: strides must be multiples of 4 elements", who);
    if (((uintptr_t)d->q | (uintptr_t)d->out) & 15) return fail(FBLT_ERR_ARG, "%s: buffers must be 16-byte aligned", who);
    return FBLT_OK;
}

// ---- plan: tile of rows and pieces of the key range --------------------------------------------------------------

int launch_paged_chunk(const PagedAttnParams &p, int hd, bool e4, cudaStream_t s); // paged_chunk.cu
int chunk_take_error();

struct PagedPlan {
    bool chunk; // the tcgen05 kernel
    int rb, wr, row_tiles, splits;
    size_t need;
};

static PagedPlan paged_plan(const fblt_paged_attn_desc *d) {
    PagedPlan pl;
    const int64_t rows = (int64_t)d->max_new * (d->num_heads / d->cache.num_kv_heads);
    const int64_t units = (int64_t)d->batch * d->cache.num_kv_heads;
    int64_t s = d->splits;
    // 64 caches of 1.5 to 8 k keys, 8 kv heads, head_dim 64 / 128: 32 rows 266 / 426 us streamed, 395 / 623 us as a chunk;
    // 48 rows 406 / 731 us and 401 / 647 us (a streaming CTA's warps each read all keys once more for every 8 or 16 rows).
    pl.chunk = rows > 32;
    if (pl.chunk) {
        pl.rb = pl.wr = 0;
        pl.row_tiles = (int)((rows + 255) / 256);
        if (s == 0) {
            // One CTA an SM: the number of pieces (of at least 1024 keys) that leaves the fewest SMs idle in the last wave;
            // one, where tiles of a sequence are three waves by themselves (a prompt of 8 k rows x 16 heads, 512 CTAs, in
            // 1 / 2 / 4 pieces: 346 / 400 / 467 us; ragged chunks 324 / 332 / 385 us; 2048 rows behind 30 k keys, 128
            // CTAs, in 1 / 8 pieces: 672 / 646 us).
            const int64_t most = pl.row_tiles > 1 && units * pl.row_tiles >= kPlanSms * 3 ? 1 : 8;
            double best = 0.0;
            for (int64_t c = 1; c <= most && (c == 1 || d->max_len / c >= 1024); ++c) {
                const int64_t ctas = units * pl.row_tiles * c, waves = (ctas + kPlanSms - 1) / kPlanSms;
                const double use = (double)ctas / (double)(waves * kPlanSms) - 0.01 * (double)(c - 1);
                if (use > best) {
                    best = use;
                    s = c;
                }
            }
        }
    } else {
        // Two blocks of 8 rows a warp while their output (64 registers a block at head_dim 128) leaves room for more than
        // one CTA on an SM: at 128 one block (two of them took 708 us where one took 557, before the sums
        // moved to shared memory).
        pl.rb = rows <= 8 || d->cache.head_dim == 128 ? 1 : 2;
        pl.wr = rows <= 8 * pl.rb ? 1 : rows <= 16 * pl.rb ? 2 : 4; // 4: head_dim 128 alone, 17 .. 32 rows
        pl.row_tiles = 1;
        if (s == 0) {
            // The GPU is filled first, as long as a piece is worth a few stages; sequences of different lengths then want
            // many times as many CTAs as run at once, as long as a piece has 512 KB of keys and values. Blocks of 8 rows x
            // 4 heads over 64 caches of 1.5 to 8 k keys, head_dim 128, in 1 / 2 / 4 / 8 pieces: 526 / 444 / 414 / 424 us;
            // 512 pieces of head_dim 64: 160 / 143 / 147 / 174 us; one token over 4 k keys: 55 / 59 us in 1 / 2 pieces.
            const int64_t ctas = units, key_max = d->max_len, worth = 256 * 1024 / d->cache.head_dim;
            const int64_t fill = std::min((int64_t)kPlanSms * 4 / ctas, key_max / 256);
            const int64_t even = std::min(((int64_t)kPlanSms * 14 + ctas - 1) / ctas, key_max / worth);
            s = std::max(fill, even);
        }
    }
    pl.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    pl.need = pl.splits > 1 ? (size_t)d->total_rows * d->num_heads * pl.splits * (d->cache.head_dim + 4) * sizeof(float) : 0;
    return pl;
}

static int paged_plan_check(const fblt_paged_attn_desc *d, const PagedPlan &pl, const void *workspace, size_t workspace_bytes) {
    if (pl.need > 0) {
        if (!workspace || workspace_bytes < pl.need)
            return fail(FBLT_ERR_WORKSPACE, "paged_attn: %zu bytes of workspace needed (fblt_paged_attn_workspace), got %zu", pl.need,
                        workspace_bytes);
        if ((uintptr_t)workspace & 15) return fail(FBLT_ERR_ARG, "paged_attn: workspace must be 16-byte aligned");
    }
    // A tile of every sequence is launched for every tile that max_new allows: beyond this many, nearly all of them empty, a
    // launch would only take milliseconds to find that out.
    const int64_t units = (int64_t)d->batch * pl.row_tiles;
    if (units >= (1 << 22) || units * pl.splits * d->cache.num_kv_heads > INT_MAX)
        return fail(FBLT_ERR_LIMIT, "paged_attn: batch * row tiles (%d) exceed 2^22 - 1, or with %d pieces and the kv heads 2^31 - 1, per launch",
                    pl.row_tiles, pl.splits);
    if (pl.splits > 1 && (int64_t)d->total_rows * d->num_heads * (d->cache.head_dim / 4) / 256 >= INT_MAX)
        return fail(FBLT_ERR_LIMIT, "paged_attn: too many rows to merge in one launch");
    return FBLT_OK;
}

// Everything that fblt_paged_attn refuses a call for, for a caller that launches other work before it.
int paged_attn_check_call(const fblt_paged_attn_desc *d, const void *workspace, size_t workspace_bytes) {
    const int st = paged_attn_check(d);
    if (st != FBLT_OK || d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return st;
    return paged_plan_check(d, paged_plan(d), workspace, workspace_bytes);
}

template <int HD, int FMT, int RB, int WR>
static int launch_stream_t(const PagedAttnParams &p, cudaStream_t s) {
    constexpr int smem = PsCta<HD, RB, WR>::kBytes;
    static_assert(4 / WR * 8 * RB * WR * (HD + 4) * 4 <= PsCta<HD, RB, WR>::kStages * PsShape<HD>::kStage, "the merge area fits the ring");
    static std::atomic<uint64_t> done{0};
    if (const int st = allow_smem((const void *)paged_stream_kernel<HD, FMT, RB, WR>, smem, done)) return st;
    paged_stream_kernel<HD, FMT, RB, WR><<<paged_grid(p), WR == 1 ? 128 : 160, smem, s>>>(p);
    count_launch();
    return check_launch("paged_stream_kernel");
}

template <int HD>
static int launch_paged(const PagedAttnParams &p, const PagedPlan &pl, bool e4, cudaStream_t s) {
    constexpr int B = HD == 128 ? 1 : 2;
    int st;
    if (pl.chunk) st = launch_paged_chunk(p, HD, e4, s);
#define FBLT_PS(RB, WR) (e4 ? launch_stream_t<HD, FBLT_KV_E4M3, RB, WR>(p, s) : launch_stream_t<HD, FBLT_KV_INT8, RB, WR>(p, s))
    else if (pl.rb == 1 && pl.wr == 1) st = FBLT_PS(1, 1);
    else if (pl.wr == 1) st = FBLT_PS(B, 1);
    else if (pl.wr == 2) st = FBLT_PS(B, 2);
    else st = FBLT_PS(B, B == 1 ? 4 : 2); // 17 .. 32 rows: four warps of one block, or (the case before) two of two
#undef FBLT_PS
    if (st != FBLT_OK || p.splits <= 1) return st;
    const int64_t units = (int64_t)p.total * p.H, per = 256 / (HD / 4);
    paged_merge_kernel<HD><<<(unsigned)((units + per - 1) / per), 256, 0, s>>>(p);
    count_launch();
    return check_launch("paged_merge_kernel");
}

int paged_take_error() {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_paged_error, sizeof(v)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_paged_error, &zero, sizeof(zero));
    const int c = chunk_take_error();
    return v ? (int)v : c;
}

} // namespace fblt

extern "C" size_t fblt_paged_attn_workspace(const fblt_paged_attn_desc *d) {
    if (fblt::paged_attn_check(d) != FBLT_OK || d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return 0;
    return fblt::paged_plan(d).need;
}

extern "C" int fblt_paged_attn(const fblt_paged_attn_desc *d, void *workspace, size_t workspace_bytes, void *stream) {
    fblt::NvtxRange nvtx_range("fblt_paged_attn");
    using namespace fblt;
    int st = paged_attn_check(d);
    if (st != FBLT_OK) return st;
    if (d->batch == 0 || d->total_rows == 0 || d->max_new == 0) return FBLT_OK;
    const PagedPlan pl = paged_plan(d);
    if ((st = paged_plan_check(d, pl, workspace, workspace_bytes)) != FBLT_OK) return st;
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
    p.splits = pl.splits;
    p.row_tiles = pl.row_tiles;
    p.cu = d->cu_new;
    p.base = d->base_len;
    p.q = d->q;
    p.qs = d->q_stride;
    p.out = d->out;
    p.os = d->out_stride;
    p.ws = (float *)workspace;
    p.qscale = d->scale * kLog2e;
    cudaStream_t s = (cudaStream_t)stream;
    const bool e4 = d->cache.format == FBLT_KV_E4M3;
    switch (d->cache.head_dim) {
    case 32: return launch_paged<32>(p, pl, e4, s);
    case 64: return launch_paged<64>(p, pl, e4, s);
    default: return launch_paged<128>(p, pl, e4, s);
    }
}
