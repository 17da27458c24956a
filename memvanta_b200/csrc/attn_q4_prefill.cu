// attn_q4_prefill.cu -- attention of chunks of query rows over the 4-bit paged
// cache on the 5th-generation tensor cores.
//
// A CTA takes NQ tiles of 128 (query row, head) pairs of one sequence and kv
// head -- 128 / G rows of its G heads -- and walks the sequence's tokens in tiles
// of NT.  Roles:
//   NQ x 4 softmax warps (thread = row of its tile = TMEM lane): queries into
//     shared memory once; then per token tile scores from TMEM, running maximum and
//     sum, weights back into TMEM;
//   4 warps that expand the cache: keys to fp16, values to tf32, both exact;
//   1 warp whose first lane issues the MMAs:
//     S (128 x NT) = Q K^T, kind::f16, Q and K from shared memory;
//     O (128 x HD) += P V, kind::tf32, P from TMEM, V from shared memory.
// A key is (n - 8) d 2^e in fp16, e per token tile such that its largest scale
// is near 2^7 (smaller scales stay exact down to 2^-20 of it).  Values and weights
// are tf32, whose exponent range no weight or scale leaves; the value of nibble
// i carries a factor 16^(i % 4) (kv_q4.cuh), taken off the columns of O at the
// end.  fp32 queries and their weights go in as two parts of 11 bits each (two
// MMAs); a half-precision query is one part, and so are its weights, cut to 11
// bits by the tensor core, with 1 + 2^-12 on them for what the cut takes off
// on average.
// A masked weight is 0, and 0 times a value that is not finite would not be: such
// value blocks enter as zeros, and the rows that see one get NaN in its
// dimensions at the end.
// Every wait is bounded (tc.cuh).
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "kv_q4.cuh"
#include "tc.cuh"

namespace mvb {

__device__ int g_q4_status = 0;  // site of an expired bounded wait (0: none)

// Adds this kernel's status to *status (first site wins) and clears it.
cudaError_t q4_status_take(int* status) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_q4_status, sizeof(int));
    if (e == cudaSuccess && v != 0) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_q4_status, &zero, sizeof(int));
        if (!*status) *status = v;
    }
    return e;
}

namespace {

constexpr int kRows = 128;  // of a query tile: TMEM lanes
constexpr int kRing = 4;    // tiles whose exponent and token masks are kept

template <int HD, int NQ, bool TWO>
struct Pf {
    static constexpr int NT = HD == 256 ? 32 : 64;  // tokens of a tile
    static constexpr int NB = HD / 32;
    static constexpr int kParts = TWO ? 2 : 1;
    static constexpr int kQ = HD / 64 * kRows * 128;   // bytes of one part of one query tile
    static constexpr int kK = HD / 64 * NT * 128;      // keys: chunks of 64 dims, a row of 128 B per token
    static constexpr int kV = NT / 32 * HD * 128;      // values: chunks of 32 tokens, a row of 128 B per dim
    static constexpr int kOffK = NQ * kParts * kQ;
    static constexpr int kOffV = kOffK + 2 * kK;
    static constexpr int kOffBar = kOffV + 2 * kV;
    // barriers: k_full, k_empty, v_full, v_empty [2]; s_full, p_full, o_done [NQ]; last
    static constexpr int kBars = 8 + 3 * NQ + 1;
    static constexpr int kOffMisc = kOffBar + kBars * 8;
    // factor 2^-e [kRing], token masks [kRing][2], blocks that are not finite: any
    // [kRing][2], which tokens [kRing][2][NB]; TMEM base, abort flag, tokens
    static constexpr int kSmem = kOffMisc + kRing * (4 + 8 + 8 + 8 * NB) + 12 + 1024;
    static constexpr int kThreads = NQ * 128 + 128 + 32;
    // TMEM columns of a query tile: scores, then weights (fp32 queries: the first
    // part in the scores' place, the second beside it), then outputs
    static constexpr int kCols = 2 * NT + HD;
    static constexpr uint32_t kTmem = NQ * kCols <= 256 ? 256 : 512;
    static_assert(NQ * kCols <= 512, "tensor memory");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct PfArgs {
    AttnQ4Args a;
    int rpt;       // query rows per tile
    int heads;     // query heads of a tile (rpt * heads <= 128)
    int chunks;    // tiles of heads per kv head
    int q_tiles;   // CTAs along a sequence's rows
    uint32_t page_mul;
    int page_shift;
};

// Instruction descriptors: both operands K-major, D f32.
__host__ __device__ constexpr uint32_t idesc(int kind_ab, int M, int N) {
    return (1u << 4) | ((uint32_t)kind_ab << 7) | ((uint32_t)kind_ab << 10) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void mma_tf32_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b), "r"(id), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
// 16-byte unit u (0..7) of row r of a 128-byte-swizzled tile
__device__ __forceinline__ uint32_t sw128(int r, int u) { return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4)); }

template <class T, int HD, int NQ>
__global__ void __launch_bounds__(Pf<HD, NQ, sizeof(T) == 4>::kThreads, 1) attn_q4_prefill_kernel(PfArgs p) {
    constexpr bool kTwo = sizeof(T) == 4;
    using C = Pf<HD, NQ, kTwo>;
    constexpr int NT = C::NT, NB = C::NB;
    extern __shared__ uint8_t raw_smem[];
    uint8_t* sm = raw_smem + ((1024 - (tc::smem_u32(raw_smem) & 1023)) & 1023);
    const uint32_t sb = tc::smem_u32(sm);
    const AttnQ4Args& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, H = (int)a.n_head_kv, G = (int)(a.n_head / a.n_head_kv);

    // ---- which tile: the last query tiles first, they see the most tokens
    const int per = (int)a.n_seq * H * p.chunks;
    const int qt = p.q_tiles - 1 - (int)(blockIdx.x / (unsigned)per);
    int rest = (int)(blockIdx.x % (unsigned)per);
    const int chunk = rest % p.chunks;
    rest /= p.chunks;
    const int kvh = rest % H, seq = rest / H;
    const int64_t seq0 = min(max(a.q_start[seq], 0), (int)a.n_q), seq1 = min(max(a.q_start[seq + 1], 0), (int)a.n_q);
    const int64_t row0 = seq0 + (int64_t)qt * NQ * p.rpt;
    if (row0 >= seq1) return;
    const int h0 = kvh * G + chunk * p.heads, nh = min(p.heads, G - chunk * p.heads);

    const uint32_t bars = sb + C::kOffBar;
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto s_full = [&](int q) { return bars + 64 + 8 * q; };
    auto p_full = [&](int q) { return bars + 64 + 8 * (NQ + q); };
    auto o_done = [&](int q) { return bars + 64 + 8 * (2 * NQ + q); };
    const uint32_t last_bar = bars + 64 + 8 * 3 * NQ;
    float* k_back = reinterpret_cast<float*>(sm + C::kOffMisc);                    // [kRing] 2^-e
    uint32_t* there = reinterpret_cast<uint32_t*>(sm + C::kOffMisc + 4 * kRing);   // [kRing][2]
    uint32_t* any_bad = there + 2 * kRing;                                         // [kRing][2]
    uint32_t* bad_tokens = any_bad + 2 * kRing;                                    // [kRing][2][NB]
    uint32_t* tmem_at = bad_tokens + 2 * kRing * NB;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_at + 1);
    int* most = reinterpret_cast<int*>(tmem_at + 2);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(k_full(i), 128);
            tc::mbar_init(v_full(i), 128);
            tc::mbar_init(k_empty(i), 1);
            tc::mbar_init(v_empty(i), 1);
        }
        for (int q = 0; q < NQ; ++q) {
            tc::mbar_init(s_full(q), 2);  // the MMAs' commit, and their issuer
            tc::mbar_init(p_full(q), 128);
            tc::mbar_init(o_done(q), 1);
        }
        tc::mbar_init(last_bar, 1);
        tc::mbar_fence_init();
        *abort_flag = 0;
        *most = 0;
    }
    constexpr int kMmaWarp = NQ * 4 + 4;
    if (warp == kMmaWarp) {
        tc::tmem_alloc(tc::smem_u32(tmem_at), C::kTmem);
        tc::tmem_relinquish();
    }
    __syncthreads();

    // ---- queries: thread m of tile q holds row m / nh, head m % nh
    const int q_of = warp / 4, m = (warp % 4) * 32 + lane;
    int ctx = 0;
    int64_t my_row = -1;
    int my_head = 0;
    float c_row = 0.0f;
    if (warp < NQ * 4) {
        const int64_t r = row0 + q_of * p.rpt + m / nh;
        if (m / nh < p.rpt && r < seq1) {
            my_row = r;
            my_head = h0 + m % nh;
            ctx = max(0, min(a.ctx_len[r], (int)a.max_ctx));
        }
        const T* src = static_cast<const T*>(a.q) + max(my_row, (int64_t)0) * (int64_t)a.q_stride + (int64_t)my_head * HD;
        float mx = 0.0f;
#pragma unroll 4
        for (int u = 0; u < HD / 8; ++u) {
            float x[8];
            load_n<8, true>(src + 8 * u, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[i]));
        }
        // times 2^e: the largest below 2^15
        const int e = max(-100, min(100, 14 - ((int)(__float_as_uint(mx) >> 23) - 127)));
        const float up = my_row >= 0 ? pow2i(e) : 0.0f;
        c_row = fmaxf(a.scale * 1.44269504088896341f * pow2i(-e), 1e-37f);
        uint8_t* dst = sm + q_of * C::kParts * C::kQ;
#pragma unroll 2
        for (int u = 0; u < HD / 8; ++u) {
            float x[8], lo[8];
            load_n<8, true>(src + 8 * u, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = my_row >= 0 ? x[i] * up : 0.0f;
                lo[i] = x[i] - __half2float(__float2half_rn(x[i]));
            }
            // dims of a unit in the order of the expanded keys: 0 4 1 5 2 6 3 7
            uint8_t* at = dst + (u / 8) * kRows * 128 + sw128(m, u % 8);
            *reinterpret_cast<uint4*>(at) = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1], x[5]),
                                                       pack_half2(x[2], x[6]), pack_half2(x[3], x[7]));
            if constexpr (kTwo)
                *reinterpret_cast<uint4*>(at + C::kQ) = make_uint4(pack_half2(lo[0], lo[4]), pack_half2(lo[1], lo[5]),
                                                                   pack_half2(lo[2], lo[6]), pack_half2(lo[3], lo[7]));
        }
        tc::fence_proxy_async_smem();
        const int top = __reduce_max_sync(0xffffffffu, ctx);
        if (lane == 0 && top) atomicMax(most, top);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_at;
    const int tokens = *most, tiles = (tokens + NT - 1) / NT;

    if (warp == kMmaWarp) {
        // ------------------------------------------------------ MMA issuer
        if (lane == 0 && tiles) {
            constexpr uint32_t id_qk = idesc(0, kRows, NT), id_pv = idesc(2, kRows, HD);
            auto wait = [&](uint32_t bar, int parity, int site) {
                return tc::mbar_wait(bar, (uint32_t)parity & 1u, abort_flag, &g_q4_status, site);
            };
            auto scores = [&](int q, int i) {
                const uint32_t kb = sb + C::kOffK + (i & 1) * C::kK, qb = sb + q * C::kParts * C::kQ;
                const uint32_t d = tmem + q * C::kCols;
#pragma unroll
                for (int part = 0; part < C::kParts; ++part)
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        mma_f16_ss(d, tc::sdesc_kmajor_sw128(qb + part * C::kQ + (k / 4) * kRows * 128) + 2 * (k % 4),
                                   tc::sdesc_kmajor_sw128(kb + (k / 4) * NT * 128) + 2 * (k % 4), id_qk, part || k);
                tc::mma_commit(s_full(q));
                tc::mbar_arrive(s_full(q));
            };
            auto outputs = [&](int q, int i) {
                const uint32_t vb = sb + C::kOffV + (i & 1) * C::kV;
                const uint32_t s = tmem + q * C::kCols, d = s + 2 * NT;
#pragma unroll
                for (int part = 0; part < C::kParts; ++part)
#pragma unroll
                    for (int k = 0; k < NT / 8; ++k)
                        mma_tf32_ts(d, s + (kTwo ? part * NT : NT) + 8 * k,
                                    tc::sdesc_kmajor_sw128(vb + (k / 4) * HD * 128) + 2 * (k % 4), id_pv,
                                    i || part || k);
                tc::mma_commit(o_done(q));
            };
            bool ok = wait(k_full(0), 0, 40);
            if (ok) {
                tc::tc_fence_after();
                for (int q = 0; q < NQ; ++q) scores(q, 0);
                tc::mma_commit(k_empty(0));
            }
            for (int i = 0; ok && i < tiles; ++i) {
                const bool more = i + 1 < tiles;
                for (int q = 0; ok && q < NQ; ++q) {
                    // the weights are in TMEM, and so the scores have been read
                    ok = wait(p_full(q), i, 41);
                    if constexpr (!kTwo) {
                        if (ok && more && q == 0) ok = wait(k_full((i + 1) & 1), (i + 1) >> 1, 42);
                        if (ok && more) {
                            tc::tc_fence_after();
                            scores(q, i + 1);
                            if (q == NQ - 1) tc::mma_commit(k_empty((i + 1) & 1));
                        }
                    }
                    if (ok && q == 0) ok = wait(v_full(i & 1), i >> 1, 43);
                    if (!ok) break;
                    tc::tc_fence_after();
                    outputs(q, i);
                    if (q == NQ - 1) tc::mma_commit(v_empty(i & 1));
                }
                if constexpr (kTwo) {
                    // the first weights' part lies where the next scores go
                    if (ok && more) ok = wait(k_full((i + 1) & 1), (i + 1) >> 1, 44);
                    for (int q = 0; ok && more && q < NQ; ++q) {
                        ok = wait(o_done(q), i, 45);
                        if (!ok) break;
                        tc::tc_fence_after();
                        scores(q, i + 1);
                        if (q == NQ - 1) tc::mma_commit(k_empty((i + 1) & 1));
                    }
                }
            }
            // every MMA issued has completed before TMEM is released
            tc::mma_commit(last_bar);
            tc::mbar_wait(last_bar, 0, abort_flag, &g_q4_status, 46, false);
        }
    } else if (warp >= NQ * 4) {
        // ------------------------------------------------ cache expansion
        constexpr int kGroups = NT / 32, kSplit = 4 / kGroups;  // warps per 32 tokens
        constexpr int W = HD / 8 / kSplit;                      // words of a token that a lane takes
        const int w4 = warp - NQ * 4, grp = w4 % kGroups, first = w4 / kGroups * W;
        const int32_t* table = a.block_table + (int64_t)seq * (int64_t)a.max_pages;
        const uint32_t page = (uint32_t)a.page;
        static_assert(W % NB == 0, "a lane's word k is of block k % NB");
        // this lane's words, its token's scales, the other group's key scales
        uint32_t kw[W], vw[W], ks[NB / 2], vs[NB / 2], ks_other[NB / 2], mask;
        auto slot_of = [&](uint32_t tok, bool& ok) -> uint64_t {
            ok = false;
            if (tok >= (uint32_t)tokens) return 0;
            const uint32_t pi = __umulhi(tok << 1, p.page_mul) >> p.page_shift, pg = (uint32_t)table[pi];
            ok = pg < (uint32_t)a.n_pages;
            return ok ? (pg * (uint32_t)H + (uint32_t)kvh) * page + (tok - pi * page) : 0;
        };
        auto scales = [&](const uint16_t* pool, uint64_t slot, bool ok, uint32_t (&out)[NB / 2]) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(pool) + slot * (NB / 2);
#pragma unroll
            for (int k = 0; k < NB / 2; ++k) out[k] = ok ? src[k] : 0u;
        };
        auto fetch = [&](int i) {
            bool ok;
            uint64_t slot = slot_of((uint32_t)i * NT + 32 * grp + lane, ok);
            mask = __ballot_sync(0xffffffffu, ok);
            scales(a.k_scales, slot, ok, ks);
            scales(a.v_scales, slot, ok, vs);
            const uint8_t* kp = a.k_pages + slot * (HD / 2) + first * 4;
            const uint8_t* vp = a.v_pages + slot * (HD / 2) + first * 4;
#pragma unroll
            for (int k = 0; k < W; k += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(kp + 4 * k);
                const uint4 y = *reinterpret_cast<const uint4*>(vp + 4 * k);
                kw[k] = x.x, kw[k + 1] = x.y, kw[k + 2] = x.z, kw[k + 3] = x.w;
                vw[k] = y.x, vw[k + 1] = y.y, vw[k + 2] = y.z, vw[k + 3] = y.w;
            }
            if constexpr (kGroups == 2) {
                slot = slot_of((uint32_t)i * NT + 32 * (grp ^ 1) + lane, ok);
                scales(a.k_scales, slot, ok, ks_other);
            }
        };
        auto scale = [](const uint32_t (&sc)[NB / 2], int b) {
            return __uint_as_float(b % 2 ? sc[b / 2] & 0xffff0000u : sc[b / 2] << 16);
        };
        auto finite = [](uint32_t bits) { return (bits & 0x7f80u) != 0x7f80u; };
        const uint64_t bias0 = held_pair(-8388616.0f, -8388736.0f), bias1 = held_pair(-8390656.0f, -8421376.0f);
        uint32_t lane_at[8];  // of this lane's token in row d of the values, d % 8 = i
#pragma unroll
        for (int i = 0; i < 8; ++i) lane_at[i] = (uint32_t)((((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
        bool ok = true;
        if (tiles) fetch(0);
        for (int i = 0; i < tiles; ++i) {
            const int s = i & 1;
            // ---- keys
            uint32_t dm = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const uint32_t x = (ks[k / 2] >> (k % 2 * 16)) & 0x7fffu;
                dm = max(dm, finite(x) ? x : 0u);
                if constexpr (kGroups == 2) {
                    const uint32_t y = (ks_other[k / 2] >> (k % 2 * 16)) & 0x7fffu;
                    dm = max(dm, finite(y) ? y : 0u);
                }
            }
            dm = __reduce_max_sync(0xffffffffu, dm);
            const int e = max(-126, min(126, 6 - ((int)(dm >> 7) - 127)));
            const float up = pow2i(e);
            ok = __all_sync(0xffffffffu, tc::mbar_wait(k_empty(s), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, &g_q4_status, 47));
            if (!ok) break;
            uint8_t* kd = sm + C::kOffK + s * C::kK;
            const int row = grp * 32 + lane;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const int t = first / NB + k / NB, b = k % NB;
                const float d = scale(ks, b) * up;
                const __half2 d2 = __float2half2_rn(d), d16 = __float2half2_rn(d * 0.0625f);
                auto mul = [](uint32_t x, __half2 y) {
                    const __half2 r = __hmul2(reinterpret_cast<const __half2&>(x), y);
                    return reinterpret_cast<const uint32_t&>(r);
                };
                const uint32_t x = kw[k], x8 = x >> 8;
                *reinterpret_cast<uint4*>(kd + (b / 2) * NT * 128 + sw128(row, (b % 2) * 4 + t)) =
                    make_uint4(mul(nib_lo(x), d2), mul(nib_hi(x), d16), mul(nib_lo(x8), d2), mul(nib_hi(x8), d16));
            }
            // value blocks that are not finite
            uint32_t bad = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) bad |= finite(vs[b / 2] >> (b % 2 * 16)) ? 0u : 1u << b;
            const bool some = __any_sync(0xffffffffu, bad);
            if (w4 < kGroups) {
                const int at = (i % kRing) * 2 + grp;
                if (lane == 0) k_back[i % kRing] = pow2i(-e), there[at] = mask, any_bad[at] = some;
                if (some)
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t which = __ballot_sync(0xffffffffu, bad >> b & 1u);
                        if (lane == 0) bad_tokens[at * NB + b] = which;
                    }
            }
            tc::fence_proxy_async_smem();
            tc::mbar_arrive(k_full(s));
            // ---- values
            ok = __all_sync(0xffffffffu, tc::mbar_wait(v_empty(s), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, &g_q4_status, 48));
            if (!ok) break;
            uint8_t* vd = sm + C::kOffV + s * C::kV + grp * HD * 128;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const int t = first / NB + k / NB, b = k % NB;
                const float d = bad >> b & 1u ? 0.0f : scale(vs, b);
                uint8_t* dst = vd + (32 * b + 8 * t) * 128;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t x = half ? vw[k] >> 16 : vw[k];
                    float v[4];
                    values2<0>(x, bias0, v[0], v[1]);
                    values2<2>(x, bias1, v[2], v[3]);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        *reinterpret_cast<float*>(dst + (half * 4 + n) * 128 + lane_at[half * 4 + n]) = v[n] * d;
                }
            }
            tc::fence_proxy_async_smem();
            tc::mbar_arrive(v_full(s));
            if (i + 1 < tiles) fetch(i + 1);
        }
    } else {
        // ------------------------------------------------------- softmax
        const uint32_t tm = tmem + q_of * C::kCols + ((uint32_t)(warp % 4) << 21);  // this warp's 32 lanes
        float m_run = -INFINITY, l = 0.0f;
        uint32_t bad = 0;  // blocks of dimensions in which this row sees values that are not finite
        bool ok = true;
        for (int i = 0; ok && i < tiles; ++i) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(s_full(q_of), (uint32_t)i & 1u, abort_flag, &g_q4_status, 49));
            if (!ok) break;
            tc::tc_fence_after();
            uint32_t s[NT / 32][32];
#pragma unroll
            for (int j = 0; j < NT / 32; ++j) tc::tmem_ld32(tm + 32 * j, s[j]);
            tc::tmem_wait_ld();
            const float c = c_row * k_back[i % kRing];
            const int left = ctx - i * NT;  // of this row's tokens
            bool cut = left < NT;
            uint32_t msk[NT / 32];  // tokens that this row sees
#pragma unroll
            for (int j = 0; j < NT / 32; ++j) {
                msk[j] = there[(i % kRing) * 2 + j];
                const int n = min(32, max(0, left - 32 * j));
                msk[j] &= n == 32 ? 0xffffffffu : (1u << n) - 1u;
                cut = cut || msk[j] != 0xffffffffu;
            }
            if (__any_sync(0xffffffffu, cut)) {
#pragma unroll
                for (int j = 0; j < NT / 32; ++j)
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!(msk[j] >> k & 1u)) s[j][k] = 0xff800000u;
            }
            for (int j = 0; j < NT / 32; ++j)
                if (any_bad[(i % kRing) * 2 + j])
                    for (int b = 0; b < NB; ++b)
                        if (bad_tokens[((i % kRing) * 2 + j) * NB + b] & msk[j]) bad |= 1u << b;
            float mx = __uint_as_float(s[0][0]);
#pragma unroll
            for (int j = 0; j < NT / 32; ++j)
#pragma unroll
                for (int k = 0; k < 32; ++k) mx = fmaxf(mx, __uint_as_float(s[j][k]));
            mx *= c;
            // the weights of the tile before have been multiplied: their place
            // is free, and the outputs may be touched
            if (i) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done(q_of), (uint32_t)(i - 1) & 1u, abort_flag, &g_q4_status, 50));
                if (!ok) break;
                tc::tc_fence_after();
            }
            // the reference m follows the maximum once that is 2^8 above it
            if (__any_sync(0xffffffffu, mx > m_run + 8.0f)) {
                const bool mine = mx > m_run + 8.0f;
                const float alpha = mine ? ex2(m_run - mx) : 1.0f;
                if (mine) m_run = mx;
                l *= alpha;
                if (i) {
#pragma unroll 1
                    for (int j = 0; j < HD / 32; ++j) {
                        uint32_t o[32];
                        tc::tmem_ld32(tm + 2 * NT + 32 * j, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tc::tmem_st32(tm + 2 * NT + 32 * j, o);
                    }
                }
            }
            // half-precision queries: weights 1 + 2^-12 larger, taken off the sum below
            const float m_use = (m_run == -INFINITY ? 0.0f : m_run) - (kTwo ? 0.0f : 3.52176e-4f);
#pragma unroll
            for (int j = 0; j < NT / 32; ++j) {
                uint32_t w[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const float pr = ex2(fmaf(__uint_as_float(s[j][k]), c, -m_use));
                    l += pr;
                    if constexpr (kTwo) {
                        const uint32_t hi = __float_as_uint(pr) & 0xffffe000u;  // 11 bits
                        w[k] = __float_as_uint(pr - __uint_as_float(hi));
                        s[j][k] = hi;
                    } else {
                        s[j][k] = __float_as_uint(pr);
                    }
                }
                tc::tmem_st32(tm + (kTwo ? 0 : NT) + 32 * j, s[j]);
                if constexpr (kTwo) tc::tmem_st32(tm + NT + 32 * j, w);
            }
            tc::tmem_wait_st();
            tc::tc_fence_before();
            tc::mbar_arrive(p_full(q_of));
        }
        // ---- outputs
        if (ok && tiles) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done(q_of), (uint32_t)(tiles - 1) & 1u, abort_flag, &g_q4_status, 51));
            tc::tc_fence_after();
        }
        if (ok) {
            const float inv = l == 0.0f ? 0.0f : (kTwo ? 1.0f : 1.000244140625f) / l;
            T* out = static_cast<T*>(a.out) + max(my_row, (int64_t)0) * (int64_t)a.out_stride + (int64_t)my_head * HD;
#pragma unroll 1
            for (int j = 0; j < HD / 32; ++j) {
                uint32_t o[32];
                if (tiles) {
                    tc::tmem_ld32(tm + 2 * NT + 32 * j, o);
                    tc::tmem_wait_ld();
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        constexpr float place[4] = {1.0f, 1.0f / 16, 1.0f / 256, 1.0f / 4096};
                        y[k] = tiles ? __uint_as_float(o[8 * u + k]) * place[k % 4] * inv : 0.0f;
                        if (bad >> j & 1u) y[k] = __uint_as_float(0x7fc00000u);
                    }
                    if (my_row >= 0) store_n<8, true>(out + 32 * j + 8 * u, y);
                }
            }
        }
    }

    // teardown: every role is out of its loop and the MMAs have drained
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        __syncwarp();
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, C::kTmem);
    }
}

template <class T, int HD, int NQ>
cudaError_t launch_prefill(PfArgs p, cudaStream_t s) {
    using C = Pf<HD, NQ, sizeof(T) == 4>;
    p.q_tiles = (int)((p.a.max_q + (uint64_t)(NQ * p.rpt) - 1) / (uint64_t)(NQ * p.rpt));
    const uint64_t grid = (uint64_t)p.q_tiles * p.a.n_seq * p.a.n_head_kv * (uint64_t)p.chunks;
    if (grid > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    auto kernel = attn_q4_prefill_kernel<T, HD, NQ>;
    ensure_smem_attr(kernel, C::kSmem);
    kernel<<<(unsigned)grid, C::kThreads, C::kSmem, s>>>(p);
    return cudaGetLastError();
}

template <class T>
cudaError_t prefill_of(const PfArgs& p, cudaStream_t s) {
    // two query tiles to a CTA share each expanded tile of the cache, where that
    // still gives every SM a CTA
    const uint64_t units = p.a.n_seq * p.a.n_head_kv * (uint64_t)p.chunks;
    const bool two = ((p.a.max_q + (uint64_t)(2 * p.rpt) - 1) / (uint64_t)(2 * p.rpt)) * units >= 148;
    if (p.a.hd == 64) return two ? launch_prefill<T, 64, 2>(p, s) : launch_prefill<T, 64, 1>(p, s);
    if (p.a.hd == 128) return two ? launch_prefill<T, 128, 2>(p, s) : launch_prefill<T, 128, 1>(p, s);
    return launch_prefill<T, 256, 1>(p, s);
}

}  // namespace

cudaError_t attn_q4_prefill(int type, const AttnQ4Args& a, cudaStream_t s) {
    PfArgs p{};
    p.a = a;
    const uint64_t G = a.n_head / a.n_head_kv;
    p.heads = (int)std::min<uint64_t>(G, kRows);
    p.chunks = (int)((G + kRows - 1) / kRows);
    p.rpt = kRows / p.heads;
    int L = 0;
    while ((1ull << L) < a.page) ++L;
    p.page_mul = (uint32_t)(((1ull << (31 + L)) + a.page - 1) / a.page);
    p.page_shift = L;
    if (type == kTypeF32) return prefill_of<float>(p, s);
    if (type == kTypeF16) return prefill_of<__half>(p, s);
    return prefill_of<__nv_bfloat16>(p, s);
}

}  // namespace mvb
