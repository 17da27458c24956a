// attn_q4_prefill.cu -- attention of chunks of query rows over the 4-bit paged
// cache on the 5th-generation tensor cores.
//
// A CTA takes NQ tiles of 128 (query row, head) pairs of one sequence and kv
// head -- 128 / G rows of its G heads -- and walks the sequence's tokens in tiles
// of NT.  Roles:
//   NQ x 4 softmax warps (thread = row of its tile = TMEM lane): per token tile
//     scores from TMEM, running maximum and sum, weights back into TMEM;
//   4 or 8 warps that expand the cache: keys to fp16, values to tf32, both exact;
//   per query tile two warps that issue the MMAs:
//     S (128 x NT) = Q K^T, kind::f16, Q and K from shared memory;
//     O (128 x HD) += P V, kind::tf32, P from TMEM, V from shared memory.
// The scores of tile i + 1 are formed while tile i's weights are: two buffers.
// A key is (n - 8) d 2^e in fp16, e per token tile such that its largest scale
// is near 2^7 (smaller scales stay exact down to 2^-20 of it).  Values and weights
// are tf32, whose exponent range no weight or scale leaves; the value of nibble
// i carries a factor 16^(i % 4) (kv_q4.cuh), taken off the columns of O at the
// end.
// fp32 queries and their weights go in as two parts of 11 bits each (two
// MMAs).  The tensor core cuts its running sums to 24 bits at every MMA instead
// of rounding: summed over a whole context that takes 1.6e-8 an MMA off the
// outputs (1.5e-4 after 32,768 tokens), so for fp32 queries a tile's outputs start
// from zero and are added to the total, rounded, by the softmax warps.  The second
// parts go first: the sum is then 2^-11 of itself for half of its cuts.
// A half-precision query is one part, and so are its weights, rounded to 11 bits
// (rounded here, since the tensor core cuts: 764 -> 782 us for 2,048 rows at 16,384
// tokens; divided by the sum of the rounded weights, 796 us).  Its outputs are
// summed by the tensor core for kRunTokens tokens at a time.
// A masked weight is 0, and 0 times a value that is not finite would not be: such
// value blocks enter as zeros, and the rows that see one get NaN in its
// dimensions at the end.
// Every wait is bounded (tc.cuh).
//
// Tiles: a query tile is as high as the MMA (128 lanes of TMEM).  64 tokens (32 for
// head_dim 256) are what two buffers of scores, the outputs and, for fp32, the
// weights' second parts leave room for in TMEM; two query tiles share an expanded
// tile where that fits (half precision, head_dim up to 128) and still gives every
// SM a CTA.  The last query tiles start first: they see the most tokens.
// Measured (back-to-back launches):
//   512 rows, 32 heads x 128, fp32                          24.4 us
//   2,048 rows after 14,336, 32 heads / 8 x 128, bf16        726 us  515 GFLOP: 0.71 PFLOP/s, 0.43 of bf16
//   7 x 331 rows after 1,500, 16 heads / 4 x 256, fp16       88 us  0.21 PFLOP/s
// Bound by latency: per token tile 1.65 us (fp32), 1.17 us (half precision, head_dim
// 128; two query tiles 3.0 us), 2.5 us (head_dim 256, 32 tokens twice), of which the
// MMAs take 0.5 to 0.6 us a query tile; the rest is the chain scores - maximum -
// weights - outputs of 64 exponentials a thread and the hand-offs.  9 us (fp32) or
// 6 us (half) are launch, queries, first tile and outputs; and the last wave of
// CTAs is part empty (256 CTAs and 308 on 148 SMs).
// Tried (when the 2,048 rows took 690 us): one warp issuing all MMAs in order (870
// us), one lane polling for its warp (+8%), a single buffer of scores (fp32 +13%),
// outputs through shared memory in whole lines (1 us less at the end, 4% more in
// the loop: registers).
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
// Half-precision queries: tokens between rounded totals of the outputs, in scratch
// (tensor memory is full).  Outputs of values of one sign after 262,144 tokens are
// 5e-5 short so, and were 1.75e-3 short without, seven times fp16's rounding.  A
// total takes some 5 us of a CTA: 2,048 rows after 14,336, bf16 755 -> 770 us, and 790
// with one every 4,096 tokens (2.6e-5).
constexpr int kRunTokens = 8192;
constexpr int kRing = 4;    // tiles whose exponent and token masks are kept

template <int HD, int NQ, bool TWO>
struct Pf {
    static constexpr int NT = HD == 256 ? 32 : 64;  // tokens of a tile
    static constexpr int NB = HD / 32;
    static constexpr int kRun = kRunTokens / NT;  // tiles between rounded totals
    static constexpr int kParts = TWO ? 2 : 1;
    static constexpr int kQ = HD / 64 * kRows * 128;   // bytes of one part of one query tile
    static constexpr int kK = HD / 64 * NT * 128;      // keys: chunks of 64 dims, a row of 128 B per token
    static constexpr int kV = NT / 32 * HD * 128;      // values: chunks of 32 tokens, a row of 128 B per dim
    static constexpr int kOffK = NQ * kParts * kQ;
    static constexpr int kOffV = kOffK + 2 * kK;
    static constexpr int kOffBar = kOffV + 2 * kV;
    // barriers: k_full, k_empty, v_full, v_empty [2]; s_full, p_full, o_done [NQ][2];
    // last, t_part, t_free
    static constexpr int kBars = 8 + 6 * NQ + 3;
    static constexpr int kOffMisc = kOffBar + kBars * 8;
    // exponents of the query rows [NQ][128]; factor 2^-e [kRing], token masks
    // [kRing][2], blocks that are not finite: any [kRing][2], which tokens
    // [kRing][2][NB]; TMEM base, abort flag, most tokens of a softmax warp's rows
    static constexpr int kSmem = kOffMisc + NQ * kRows * 4 + kRing * (4 + 8 + 8 + 8 * NB) + 8 + NQ * 16 + 1024;
    static constexpr int kExpand = NQ == 2 ? 4 : 8;  // warps
    static constexpr int kThreads = NQ * 128 + kExpand * 32 + 2 * NQ * 32;
    // TMEM columns of a query tile: two buffers of NT scores, taken by the
    // weights (their first part) of the same token tile; fp32: two of the weights'
    // second part, and a tile's outputs, OT columns at a time; outputs HD.
    static constexpr int OT = HD == 256 ? 128 : HD;
    static constexpr int kOffL = 2 * NT, kOffT = 4 * NT;
    static constexpr int kOffO = TWO ? kOffT + OT : 2 * NT;
    static constexpr int kCols = kOffO + HD;
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
    // half precision, contexts longer than kRunTokens: [kv head][chunk][hd][n_q * heads], so
    // that a warp's rows, which follow one another, lie so in every column
    float* totals;
};

// Instruction descriptors: both operands K-major, D f32.
__host__ __device__ constexpr uint32_t idesc(int kind_ab, int M, int N) {
    return (1u << 4) | ((uint32_t)kind_ab << 7) | ((uint32_t)kind_ab << 10) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// The MMAs and their commit are called by a whole warp and issued by one
// elected lane of it: with operands that are the same in every lane, one takes
// some 20 cycles to issue (from a branch of one lane, 60 to 75).
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void mma_tf32_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b), "r"(id), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// 16-byte unit u (0..7) of row r of a 128-byte-swizzled tile
__device__ __forceinline__ uint32_t sw128(int r, int u) { return (uint32_t)(r * 128 + ((u ^ (r & 7)) << 4)); }

// Half-precision queries: the outputs of a run of tiles (TMEM, this warp's lanes) go
// to a row's totals, one for each column, `pairs` apart; `more`: on top of those
// of the runs before, times `keep`.  (Functions of their own: inlined, they cost
// the loop over the tiles its registers, 8% of the time.)
template <int HD>
__device__ __noinline__ void end_run(uint32_t o_at, float* total, int64_t pairs, bool more, float keep) {
#pragma unroll 1
    for (int j = 0; j < HD; j += 32) {
        uint32_t o[32];
        float y[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) y[k] = more && total ? total[(j + k) * pairs] : 0.0f;
        tc::tmem_ld32(o_at + j, o);
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k)
            if (total) total[(j + k) * pairs] = fmaf(y[k], keep, __uint_as_float(o[k]));
    }
}
// And the totals, times `keep`, to the outputs of the last run.
template <int HD>
__device__ __noinline__ void add_runs(uint32_t o_at, const float* total, int64_t pairs, float keep) {
#pragma unroll 1
    for (int j = 0; j < HD; j += 32) {
        uint32_t o[32];
        float y[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) y[k] = total ? total[(j + k) * pairs] : 0.0f;
        tc::tmem_ld32(o_at + j, o);
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(fmaf(y[k], keep, __uint_as_float(o[k])));
        tc::tmem_st32(o_at + j, o);
    }
    tc::tmem_wait_st();
}

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
    const int64_t seq0 = a.one_seq ? 0 : min(max(a.q_start[seq], 0), (int)a.n_q);
    const int64_t end = a.one_seq ? (int64_t)a.n_q : min(max(a.q_start[seq + 1], 0), (int)a.n_q);
    const int64_t seq1 = min(end, seq0 + (int64_t)a.max_q);
    const int64_t row0 = seq0 + (int64_t)qt * NQ * p.rpt;
    const int h0 = kvh * G + chunk * p.heads, nh = min(p.heads, G - chunk * p.heads);
    if (qt == p.q_tiles - 1) {  // rows of no chunk, and past max_q, are zeros
        auto zeros = [&](int64_t from, int64_t to) {
            for (int64_t r = from; r < to; ++r)
                for (int k = threadIdx.x; k < nh * HD; k += blockDim.x)
                    static_cast<T*>(a.out)[r * (int64_t)a.out_stride + (int64_t)h0 * HD + k] = T(0.0f);
        };
        zeros(seq1, end);
        if (seq == 0) zeros(0, seq0);
        if (seq == (int)a.n_seq - 1) zeros(max(seq0, end), (int64_t)a.n_q);
    }
    if (row0 >= seq1) return;

    const uint32_t bars = sb + C::kOffBar;
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto s_full = [&](int q, int i) { return bars + 64 + 8 * (2 * q + (i & 1)); };
    auto p_full = [&](int q, int i) { return bars + 64 + 8 * (2 * NQ + 2 * q + (i & 1)); };
    auto o_done = [&](int q, int i) { return bars + 64 + 8 * (4 * NQ + 2 * q + (i & 1)); };
    const uint32_t last_bar = bars + 64 + 8 * 6 * NQ, t_part = last_bar + 8, t_free = last_bar + 16;
    int* q_exp = reinterpret_cast<int*>(sm + C::kOffMisc);                         // [NQ][128]
    float* k_back = reinterpret_cast<float*>(q_exp + NQ * kRows);                  // [kRing] 2^-e
    uint32_t* there = reinterpret_cast<uint32_t*>(k_back + kRing);                 // [kRing][2]
    uint32_t* any_bad = there + 2 * kRing;                                         // [kRing][2]
    uint32_t* bad_tokens = any_bad + 2 * kRing;                                    // [kRing][2][NB]
    uint32_t* tmem_at = bad_tokens + 2 * kRing * NB;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_at + 1);
    int* most = reinterpret_cast<int*>(tmem_at + 2);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(k_full(i), C::kExpand * 32);
            tc::mbar_init(v_full(i), C::kExpand * 32);
            tc::mbar_init(k_empty(i), NQ);
            tc::mbar_init(v_empty(i), NQ);
        }
        for (int q = 0; q < NQ; ++q)
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(s_full(q, i), 2);  // the MMAs' commit, and their issuer
                tc::mbar_init(p_full(q, i), 128);
                tc::mbar_init(o_done(q, i), 1);
            }
        tc::mbar_init(last_bar, 2 * NQ);
        tc::mbar_init(t_part, 1);
        tc::mbar_init(t_free, 128);  // a tile's first OT columns are taken out
        tc::mbar_fence_init();
        *abort_flag = 0;
    }
    constexpr int kMmaWarp = NQ * 4 + C::kExpand;
    if (warp == kMmaWarp) {
        tc::tmem_alloc(tc::smem_u32(tmem_at), C::kTmem);
        tc::tmem_relinquish();
    }
    // softmax thread m of tile q holds row m of it, query m / nh, head m % nh
    const int q_of = warp / 4, m_of = (warp % 4) * 32 + lane;
    int ctx = 0, my_head = 0;
    int64_t my_row = -1;
    if (warp < NQ * 4) {
        const int64_t r = row0 + q_of * p.rpt + m_of / nh;
        if (m_of / nh < p.rpt && r < seq1) {
            my_row = r;
            my_head = h0 + m_of % nh;
            ctx = max(0, min(a.ctx_len[r], (int)a.max_ctx));
        }
        const int top = __reduce_max_sync(0xffffffffu, ctx);
        if (lane == 0) most[warp] = top;
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_at;
    int tokens = 0;
#pragma unroll
    for (int w = 0; w < NQ * 4; ++w) tokens = max(tokens, most[w]);
    const int tiles = (tokens + NT - 1) / NT;

    if (warp >= kMmaWarp) {
        // ----------------------------------------------------- MMA issuers
        // (a uniform role and tile: the MMAs' operands stay in uniform registers)
        const int role = __shfl_sync(0xffffffffu, warp - kMmaWarp, 0), q = role % NQ;
        const uint32_t t = tmem + q * C::kCols;
        auto wait = [&](uint32_t bar, int parity, int site) {
            if (!__all_sync(0xffffffffu, tc::mbar_wait(bar, (uint32_t)parity & 1u, abort_flag, &g_q4_status, site)))
                return false;
            tc::tc_fence_after();
            return true;
        };
        if (tiles) {
            if (role < NQ) {
                // scores, into the buffer whose weights, of two tiles before, have been multiplied
                constexpr uint32_t id = idesc(0, kRows, NT);
                const uint32_t qb = sb + q * C::kParts * C::kQ;
                asm volatile("bar.sync %0, 160;" ::"r"(1 + q) : "memory");  // the tile's queries are there
                for (int i = 0; i < tiles; ++i) {
                    if (!wait(k_full(i & 1), i >> 1, 40)) break;
                    if (i >= 2 && !wait(o_done(q, i), (i - 2) >> 1, 41)) break;
                    const uint32_t kb = sb + C::kOffK + (i & 1) * C::kK, d = t + (i & 1) * NT;
#pragma unroll
                    for (int part = C::kParts - 1; part >= 0; --part)
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            mma_f16_ss(d,
                                       tc::sdesc_kmajor_sw128(qb + part * C::kQ + (k / 4) * kRows * 128) + 2 * (k % 4),
                                       tc::sdesc_kmajor_sw128(kb + (k / 4) * NT * 128) + 2 * (k % 4), id,
                                       part + 1 < C::kParts || k);
                    commit(s_full(q, i));
                    if (lane == 0) tc::mbar_arrive(s_full(q, i));
                    commit(k_empty(i & 1));
                }
            } else {
                // outputs, OT columns at a time for fp32
                constexpr uint32_t id = idesc(2, kRows, kTwo ? C::OT : HD);
                constexpr int kTurns = kTwo ? HD / C::OT : 1;
                bool ok = true;
                for (int i = 0; ok && i < tiles; ++i) {
                    ok = wait(v_full(i & 1), i >> 1, 42) && wait(p_full(q, i), i >> 1, 43);
#pragma unroll
                    for (int turn = 0; turn < kTurns; ++turn) {
                        if (turn && ok) ok = wait(t_free, i, 44);  // the columns before are taken out
                        if (!ok) break;
                        const uint32_t vb = sb + C::kOffV + (i & 1) * C::kV + turn * C::OT * 128;
                        const uint32_t d = t + (kTwo ? C::kOffT : C::kOffO);
#pragma unroll
                        for (int part = C::kParts - 1; part >= 0; --part)
#pragma unroll
                            for (int k = 0; k < NT / 8; ++k)
                                mma_tf32_ts(d, t + part * C::kOffL + (i & 1) * NT + 8 * k,
                                            tc::sdesc_kmajor_sw128(vb + (k / 4) * HD * 128) + 2 * (k % 4), id,
                                            (!kTwo && i % C::kRun) || part + 1 < C::kParts || k);
                        commit(turn + 1 < kTurns ? t_part : o_done(q, i));
                    }
                    if (ok) commit(v_empty(i & 1));
                }
            }
            // every MMA issued has completed before TMEM is released
            commit(last_bar);
            tc::mbar_wait(last_bar, 0, abort_flag, &g_q4_status, 46, false);
        }
    } else if (warp >= NQ * 4) {
        // ------------------------------------------------ cache expansion
        constexpr int kGroups = NT / 32, kSplit = C::kExpand / kGroups;  // warps per 32 tokens
        constexpr int W = HD / 8 / kSplit;                               // words of a token that a lane takes
        static_assert(W % NB == 0 || NB % W == 0, "a warp's words start at a block that its lanes share");
        const int w8 = warp - NQ * 4, grp = w8 % kGroups, first = w8 / kGroups * W;
        const int b0 = first % NB, t0 = first / NB;  // block and quarter of the first word
        const int32_t* table = a.block_table + (int64_t)seq * (int64_t)a.max_pages;
        const uint32_t page = (uint32_t)a.page;
        // this lane's words, its token's scales, the other group's key scales
        struct Raw {
            uint32_t kw[W], vw[W], ks[NB / 2], vs[NB / 2], ks_other[NB / 2], mask;
        };
        // slots of this lane's token of the tile after the fetched one, looked up a tile ahead
        uint32_t slot_own = 0, slot_other = 0;
        bool ok_own = false, ok_other = false;
        auto slot_of = [&](uint32_t tok, bool& ok) -> uint32_t {
            ok = false;
            if (tok >= (uint32_t)tokens) return 0;
            const uint32_t pi = __umulhi(tok << 1, p.page_mul) >> p.page_shift, pg = (uint32_t)table[pi];
            ok = pg < (uint32_t)a.n_pages;
            return ok ? (pg * (uint32_t)H + (uint32_t)kvh) * page + (tok - pi * page) : 0;
        };
        auto look_up = [&](int i) {
            slot_own = slot_of((uint32_t)i * NT + 32 * grp + lane, ok_own);
            if constexpr (kGroups == 2) slot_other = slot_of((uint32_t)i * NT + 32 * (grp ^ 1) + lane, ok_other);
        };
        auto scales = [&](const uint16_t* pool, uint32_t slot, bool ok, uint32_t (&out)[NB / 2]) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(pool) + (uint64_t)slot * (NB / 2);
#pragma unroll
            for (int k = 0; k < NB / 2; ++k) out[k] = ok ? src[k] : 0u;
        };
        auto words = [&](const uint8_t* pool, uint32_t (&out)[W]) {
            const uint8_t* src = pool + (uint64_t)slot_own * (HD / 2) + first * 4;
            if constexpr (W == 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(src);
                out[0] = x.x, out[1] = x.y;
            } else {
#pragma unroll
                for (int k = 0; k < W; k += 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(src + 4 * k);
                    out[k] = x.x, out[k + 1] = x.y, out[k + 2] = x.z, out[k + 3] = x.w;
                }
            }
        };
        auto fetch = [&](Raw& r) {
            r.mask = __ballot_sync(0xffffffffu, ok_own);
            scales(a.k_scales, slot_own, ok_own, r.ks);
            scales(a.v_scales, slot_own, ok_own, r.vs);
            words(a.k_pages, r.kw);
            words(a.v_pages, r.vw);
            if constexpr (kGroups == 2) scales(a.k_scales, slot_other, ok_other, r.ks_other);
        };
        // scale of the block of word k
        auto scale = [&](const uint32_t (&sc)[NB / 2], int k) {
            const int b = k % NB;
            uint32_t w = sc[b / 2];
            if constexpr (W < NB) w = b0 ? sc[b / 2 + W / 2] : w;
            return __uint_as_float(b % 2 ? w & 0xffff0000u : w << 16);
        };
        auto finite = [](uint32_t bits) { return (bits & 0x7f80u) != 0x7f80u; };
        const uint64_t bias0 = held_pair(-8388616.0f, -8388736.0f), bias1 = held_pair(-8390656.0f, -8421376.0f);
        uint32_t lane_at[8];  // of this lane's token in row d of the values, d % 8 = i
#pragma unroll
        for (int i = 0; i < 8; ++i) lane_at[i] = (uint32_t)((((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
        // expands tile i from r, fetching tile i + 1 into `ahead` meanwhile
        auto expand = [&](const Raw& r, Raw& ahead, int i) -> bool {
            const int s = i & 1;
            if (i + 1 < tiles) {
                fetch(ahead);
                look_up(i + 2);
            }
            // ---- keys
            uint32_t dm = 0, bad = 0;
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const uint32_t x = (r.ks[k / 2] >> (k % 2 * 16)) & 0x7fffu;
                dm = max(dm, finite(x) ? x : 0u);
                if constexpr (kGroups == 2) {
                    const uint32_t y = (r.ks_other[k / 2] >> (k % 2 * 16)) & 0x7fffu;
                    dm = max(dm, finite(y) ? y : 0u);
                }
                bad |= finite(r.vs[k / 2] >> (k % 2 * 16)) ? 0u : 1u << k;  // value blocks that are not finite
            }
            dm = __reduce_max_sync(0xffffffffu, dm);
            const bool some = __any_sync(0xffffffffu, bad);
            // (a tile without scales, of zeros or of missing tokens: any exponent does)
            const int e = dm ? max(-126, min(126, 6 - ((int)(dm >> 7) - 127))) : 0;
            const float up = pow2i(e);
            if (!__all_sync(0xffffffffu,
                            tc::mbar_wait(k_empty(s), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, &g_q4_status, 47)))
                return false;
            uint8_t* kd = sm + C::kOffK + s * C::kK;
            const int row = grp * 32 + lane;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const int b = b0 + k % NB, t = t0 + k / NB;
                const float d = scale(r.ks, k) * up;
                const __half2 d2 = __float2half2_rn(d), d16 = __float2half2_rn(d * 0.0625f);
                auto mul = [](uint32_t x, __half2 y) {
                    const __half2 v = __hmul2(reinterpret_cast<const __half2&>(x), y);
                    return reinterpret_cast<const uint32_t&>(v);
                };
                const uint32_t x = r.kw[k], x8 = x >> 8;
                *reinterpret_cast<uint4*>(kd + (b / 2) * NT * 128 + sw128(row, (b % 2) * 4 + t)) =
                    make_uint4(mul(nib_lo(x), d2), mul(nib_hi(x), d16), mul(nib_lo(x8), d2), mul(nib_hi(x8), d16));
            }
            if (w8 < kGroups) {
                const int at = (i % kRing) * 2 + grp;
                if (lane == 0) k_back[i % kRing] = pow2i(-e), there[at] = r.mask, any_bad[at] = some;
                if (some)
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t which = __ballot_sync(0xffffffffu, bad >> b & 1u);
                        if (lane == 0) bad_tokens[at * NB + b] = which;
                    }
            }
            tc::fence_proxy_async_smem();
            tc::mbar_arrive(k_full(s));
            // ---- values
            if (!__all_sync(0xffffffffu,
                            tc::mbar_wait(v_empty(s), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, &g_q4_status, 48)))
                return false;
            uint8_t* vd = sm + C::kOffV + s * C::kV + grp * HD * 128;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const int b = b0 + k % NB, t = t0 + k / NB;
                float d = scale(r.vs, k);
                if (some && (bad >> b & 1u)) d = 0.0f;
                uint8_t* dst = vd + (32 * b + 8 * t) * 128;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t x = half ? r.vw[k] >> 16 : r.vw[k];
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
            return true;
        };
        Raw ra, rb;
        if (tiles) {
            look_up(0);
            fetch(ra);
            look_up(1);
        }
        for (int i = 0; i < tiles; i += 2) {
            if (!expand(ra, rb, i)) break;
            if (i + 1 < tiles && !expand(rb, ra, i + 1)) break;
        }
    } else {
        // ------------------------------------------------------- softmax
        // First this warp's 32 query rows, 8 lanes to a row, into shared memory (the
        // cache's first tile is fetched and expanded meanwhile)
        constexpr int kPer = HD / 64;                                        // 8-dimension units of a lane
        constexpr int kRows4 = std::min(8, (sizeof(T) == 4 ? 8 : 16) / kPer);  // times 4 rows in flight
        const int u0 = lane % 8;
#pragma unroll 1
        for (int it = 0; it < 8; it += kRows4) {
            Held<T, 8, true> in[kRows4][kPer];
            bool there_is[kRows4];
#pragma unroll
            for (int k = 0; k < kRows4; ++k) {
                const int m = (warp % 4) * 32 + (it + k) * 4 + lane / 8;
                const int64_t row = row0 + q_of * p.rpt + m / nh;
                there_is[k] = m / nh < p.rpt && row < seq1;
                const int64_t at = there_is[k] ? row * (int64_t)a.q_stride + (int64_t)(h0 + m % nh) * HD : 0;
#pragma unroll
                for (int u = 0; u < kPer; ++u) in[k][u].load(static_cast<const T*>(a.q) + at + 8 * (u0 + 8 * u));
            }
#pragma unroll
            for (int k = 0; k < kRows4; ++k) {
                const int m = (warp % 4) * 32 + (it + k) * 4 + lane / 8;
                float x[kPer][8], mx = 0.0f;
#pragma unroll
                for (int u = 0; u < kPer; ++u) {
                    in[k][u].get(x[u]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (!there_is[k]) x[u][i] = 0.0f;
                        mx = fmaxf(mx, fabsf(x[u][i]));
                    }
                }
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                // times 2^e: the largest below 2^15, whatever its size (e > 100 would take the
                // scores' factor out of range, and queries that small need no more bits)
                const int e = min(100, 14 - ((int)(__float_as_uint(mx) >> 23) - 127));
                const float up = pow2i(e);
                if (u0 == 0) q_exp[q_of * kRows + m] = e;
#pragma unroll
                for (int u = 0; u < kPer; ++u) {
                    float lo[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[u][i] *= up;
                        lo[i] = x[u][i] - __half2float(__float2half_rn(x[u][i]));
                    }
                    // dims of a unit in the order of the expanded keys: 0 4 1 5 2 6 3 7
                    uint8_t* to = sm + q_of * C::kParts * C::kQ + u * kRows * 128 + sw128(m, u0);
                    *reinterpret_cast<uint4*>(to) =
                        make_uint4(pack_half2(x[u][0], x[u][4]), pack_half2(x[u][1], x[u][5]),
                                   pack_half2(x[u][2], x[u][6]), pack_half2(x[u][3], x[u][7]));
                    if constexpr (kTwo)
                        *reinterpret_cast<uint4*>(to + C::kQ) =
                            make_uint4(pack_half2(lo[0], lo[4]), pack_half2(lo[1], lo[5]), pack_half2(lo[2], lo[6]),
                                       pack_half2(lo[3], lo[7]));
                }
            }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();  // the exponents, too
        if (tiles) asm volatile("bar.arrive %0, 160;" ::"r"(1 + q_of) : "memory");
        const uint32_t tm = tmem + q_of * C::kCols + ((uint32_t)(warp % 4) << 21);  // this warp's 32 lanes
        const float c_row = a.scale * 1.44269504088896341f * pow2i(-q_exp[q_of * kRows + m_of]);
        float m_run = -INFINITY, l = 0.0f, m_total = -INFINITY;  // m_total: reference of the totals
        const int64_t pairs = (int64_t)a.n_q * p.heads;
        float* total = nullptr;
        if constexpr (!kTwo)
            if (my_row >= 0)
                total = p.totals + (int64_t)(kvh * p.chunks + chunk) * HD * pairs + my_row * p.heads + m_of % nh;
        // what moves the totals from their reference to m (a total without tokens is zeros)
        auto total_factor = [&](float m) { return m_total == -INFINITY ? 0.0f : ex2(m_total - m); };
        uint32_t bad = 0;  // blocks of dimensions in which this row sees values that are not finite
        bool ok = true;
        auto wait = [&](uint32_t bar, int parity, int site) {
            const bool got = __all_sync(0xffffffffu,
                                        tc::mbar_wait(bar, (uint32_t)parity & 1u, abort_flag, &g_q4_status, site));
            if (got) tc::tc_fence_after();
            return got;
        };
        // fp32: adds tile i's outputs to the total, OT columns at a time
        auto add_tile = [&](int i) {
#pragma unroll 1
            for (int turn = 0; turn < HD / C::OT; ++turn) {
                if (turn + 1 < HD / C::OT ? !wait(t_part, i, 52) : !wait(o_done(q_of, i), i >> 1, 50)) return false;
#pragma unroll 1
                for (int j = 0; j < C::OT / 32; ++j) {
                    const uint32_t at = tm + C::kOffO + turn * C::OT + 32 * j;
                    uint32_t x[32], o[32];
                    tc::tmem_ld32(tm + C::kOffT + 32 * j, x);
                    if (i) tc::tmem_ld32(at, o);
                    tc::tmem_wait_ld();
                    if (i)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            x[k] = __float_as_uint(__uint_as_float(x[k]) + __uint_as_float(o[k]));
                    tc::tmem_st32(at, x);
                }
                if (turn + 1 < HD / C::OT) {  // the next columns may come
                    tc::tc_fence_before();
                    tc::mbar_arrive(t_free);
                }
            }
            tc::tmem_wait_st();
            return true;
        };
        for (int i = 0; ok && i < tiles; ++i) {
            if (!kTwo && i && i % C::kRun == 0) {
                // a run of tiles has ended: its outputs go to the totals, and the next
                // one's start from zero
                ok = wait(o_done(q_of, i - 1), (i - 1) >> 1, 53);
                if (!ok) break;
                end_run<HD>(tm + C::kOffO, total, pairs, i > C::kRun, total_factor(m_run));
                m_total = m_run;
            }
            ok = wait(s_full(q_of, i), i >> 1, 49);
            if (!ok) break;
            const uint32_t ts = tm + (i & 1) * NT;  // this tile's scores, and weights
            uint32_t s[NT / 32][32];
#pragma unroll
            for (int j = 0; j < NT / 32; ++j) tc::tmem_ld32(ts + 32 * j, s[j]);
            tc::tmem_wait_ld();
            // above zero: a masked score is -inf, and -inf * 0 would be NaN.  Scores stay
            // below 2^33 here, so a factor that small makes every one of them vanish.
            const float c = fmaxf(c_row * k_back[i % kRing], 1e-37f);
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
            // four chains each for the maximum and the sum: one is 64 dependent steps
            float mx4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) mx4[k] = __uint_as_float(s[0][k]);
#pragma unroll
            for (int j = 0; j < NT / 32; ++j)
#pragma unroll
                for (int k = 0; k < 32; ++k) mx4[k % 4] = fmaxf(mx4[k % 4], __uint_as_float(s[j][k]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * c;
            // the reference m follows the maximum once that is 2^8 above it
            const bool move = mx > m_run + 8.0f;
            const float alpha = move ? ex2(m_run - mx) : 1.0f;
            if (move) m_run = mx;
            l *= alpha;
            const float m_use = m_run == -INFINITY ? 0.0f : m_run;
            const uint64_t cc = pair(c, c), mm = pair(-m_use, -m_use);
            uint64_t l2[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < NT / 16; ++j) {
                uint32_t w[16], w2[16];
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const uint32_t* sp = &s[j / 2][j % 2 * 16 + k];
                    float x0, x1;
                    unpair(tc::f2_fma(pair(__uint_as_float(sp[0]), __uint_as_float(sp[1])), cc, mm), x0, x1);
                    x0 = ex2(x0), x1 = ex2(x1);
                    l2[k / 2 % 2] = f2_add(l2[k / 2 % 2], pair(x0, x1));
                    if constexpr (!kTwo) x0 = near11(x0), x1 = near11(x1);
                    w[k] = __float_as_uint(x0), w[k + 1] = __float_as_uint(x1);
                    if constexpr (kTwo) {
                        w[k] &= 0xffffe000u, w[k + 1] &= 0xffffe000u;  // 11 bits
                        w2[k] = __float_as_uint(x0 - __uint_as_float(w[k]));
                        w2[k + 1] = __float_as_uint(x1 - __uint_as_float(w[k + 1]));
                    }
                }
                tc::tmem_st16(ts + 16 * j, w);
                if constexpr (kTwo) tc::tmem_st16(ts + C::kOffL + 16 * j, w2);
            }
            float x0, x1;
            unpair(f2_add(l2[0], l2[1]), x0, x1);
            l += x0 + x1;
            // the outputs up to the tile before, on the new reference
            if constexpr (kTwo)
                if (i) ok = add_tile(i - 1);
            if (ok && (kTwo ? i : i % C::kRun) && __any_sync(0xffffffffu, move)) {
                if constexpr (!kTwo) ok = wait(o_done(q_of, i - 1), (i - 1) >> 1, 50);
#pragma unroll 1
                for (int j = 0; ok && j < HD / 32; ++j) {
                    uint32_t o[32];
                    tc::tmem_ld32(tm + C::kOffO + 32 * j, o);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                    tc::tmem_st32(tm + C::kOffO + 32 * j, o);
                }
            }
            if (!ok) break;
            tc::tmem_wait_st();
            tc::tc_fence_before();
            tc::mbar_arrive(p_full(q_of, i));
        }
        // ---- outputs
        if (ok && tiles) {
            if constexpr (kTwo) ok = add_tile(tiles - 1);
            else ok = wait(o_done(q_of, tiles - 1), (tiles - 1) >> 1, 51);
        }
        if (ok) {
            if (!kTwo && tiles > C::kRun) add_runs<HD>(tm + C::kOffO, total, pairs, total_factor(m_run));
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = static_cast<T*>(a.out) + max(my_row, (int64_t)0) * (int64_t)a.out_stride + (int64_t)my_head * HD;
#pragma unroll 1
            for (int j = 0; j < HD / 32; ++j) {
                uint32_t o[32];
                if (tiles) {
                    tc::tmem_ld32(tm + C::kOffO + 32 * j, o);
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
    const bool two = prefill_tiles(p.a, 2 * (uint64_t)p.rpt) * p.a.n_head_kv * (uint64_t)p.chunks >= 148;
    if constexpr (sizeof(T) == 2) {  // (fp32: tensor memory holds one)
        if (two && p.a.hd == 64) return launch_prefill<T, 64, 2>(p, s);
        if (two && p.a.hd == 128) return launch_prefill<T, 128, 2>(p, s);
    }
    if (p.a.hd == 64) return launch_prefill<T, 64, 1>(p, s);
    if (p.a.hd == 128) return launch_prefill<T, 128, 1>(p, s);
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
    if (a.max_ctx > kRunTokens) {
        const uint64_t bytes = a.n_q * a.n_head_kv * p.chunks * p.heads * a.hd * sizeof(float);
        if (cudaError_t e = scratch_alloc(reinterpret_cast<void**>(&p.totals), bytes, s)) return e;
    }
    cudaError_t e = type == kTypeF16 ? prefill_of<__half>(p, s) : prefill_of<__nv_bfloat16>(p, s);
    if (p.totals) {
        const cudaError_t f = cudaFreeAsync(p.totals, s);
        if (e == cudaSuccess) e = f;
    }
    return e;
}

}  // namespace mvb
