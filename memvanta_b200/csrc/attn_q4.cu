// attn_q4.cu -- attention over the 4-bit paged cache (kv_q4.cuh).
//
//   out[r][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[r][h].k_t - m)
// over the first ctx_len[r] cached tokens of the row's sequence, in one pass
// with the running maximum m and sum.  A row with no tokens gives zeros; what
// lies past ctx_len, or on a page that does not exist, is never used.
//
// Measured (back-to-back launches; 2 x (hd / 2 + hd / 16) bytes a token and kv head):
//   1 x 768 tokens, 32 kv heads x 128, fp32 queries          6.7 us  (latency)
//   1 x 131,071 tokens, 8 kv heads x 128, 32 heads fp32      59.1 us  151 MB: 2.6 TB/s, 0.39 of HBM's
//   64 x 64..768 tokens, 32 heads x 128 fp32                 48.3 us  1.9 TB/s
//   48 x 1..16,384 tokens, 8 kv heads x 64, 64 heads fp16    66.8 us  2.3 TB/s
//   64 x 2,000 tokens, 4 kv heads x 256, 16 heads bf16       66.4 us  2.2 TB/s
// Long contexts are bound by instructions -- some 440 for 16 tokens of head_dim 128, half
// of the integer pipe's time, a third of the tensor cores' -- and not by memory:
// the same ring without its arithmetic takes 24.5 us for the 59.1.
// Tried: two stages to a ring, 80 to 96 registers, more and smaller CTAs (slower).
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "kv_q4.cuh"
#include "tc.cuh"

namespace mvb {

namespace {

// The sequence of query row r: r itself, or by bisection of q_start (ascending);
// -1: none, or past the max_q rows that it may have.
__device__ __forceinline__ int seq_of_row(const AttnQ4Args& a, int r) {
    if (a.one_seq) return 0;
    if (!a.q_start) return r;
    if (r < a.q_start[0] || r >= a.q_start[a.n_seq]) return -1;
    int lo = 0, hi = (int)a.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.q_start[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return (uint64_t)(r - a.q_start[lo]) < a.max_q ? lo : -1;
}

// ------------------------------------------------------------- primitives
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Asynchronous copies global -> shared; `bytes` 0 fills with zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_fill(uint32_t dst, const void* src, int bytes) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes)
                     : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// D (16 x 8, fp32) = A (16 x 16, fp16) B (16 x 8, fp16) + C
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// D (16 x 8, fp32) += A (16 x 8, tf32) B (8 x 8, tf32)
__device__ __forceinline__ void mma1688(float (&d)[4], const float (&a)[4], float b0, float b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
          "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// ---------------------------------------------------------- one query row
// The work is a row of stages -- 4096 / HD tokens of one unit (a query row, a
// kv head, up to 8 of its query heads) -- cut into equal runs, one for each
// warp that the GPU holds at once, whatever the contexts' lengths.  A warp
// streams its run through a ring of its own in shared memory (cp.async; no
// barrier after the start) and goes from unit to unit without draining it.  A
// unit inside one run is written out by its warp; the parts of the others go to
// scratch and are joined by a second kernel.
//
// Both products run on the tensor cores, the cache as integers:
//  scores  (heads x tokens, m16n8k16 fp16): A = the queries, B = keys n - 8,
//          exact; each 32-block's sum is multiplied by its scale afterwards, in
//          fp32.
//  outputs (dims x heads, m16n8k8 tf32): A = values (n - 8) 16^i, exact, the
//          power of the nibble's place taken off at the end; B = the weights p d
//          with the block's scale.  tf32 keeps the weights' whole exponent
//          range: in fp16 a dimension whose heavy tokens are all zero lost the
//          light ones.
// fp32 queries and their weights go in as two parts of 11 bits: the queries'
// second parts are rows 8..15 of A, the weights' are columns 4..7 for up to
// four heads (PACK: rows 4..7 repeat heads 0..3, so a lane's weights are
// already there) and a second MMA for more.  The tensor core ignores the low
// 13 bits of a tf32 operand, so the first part needs no masking; half-precision
// queries' weights go in as one part, rounded to 11 bits.
constexpr int kWarps = 4, kStages = 3;
constexpr int kShort = 8;  // stages to a warp of a cluster at most

template <int HD>
struct Q4Tile {
    static constexpr int TT = 4096 / HD;  // tokens of a stage: 2 KB of keys, 2 KB of values
    static constexpr int NB = HD / 32;    // scale blocks
    static constexpr int U = HD / 32;     // 16-byte units of a token's nibbles
    static constexpr int NJ = TT / 8;     // 8-token fragments
    static constexpr int kScale = TT * NB * 2;
    static constexpr int kBytes = 2 * 2048 + 2 * kScale;  // K, V, K scales, V scales
    static constexpr int kRing = kStages * kBytes;
    // a warp's outputs so far, 16 x 8 per 16 dimensions (both parts), and the references that they are on
    static constexpr int kTotal = HD * 8 * 4 + 32 * 4;
    static constexpr int kFlush = 32 / NJ;  // stages between their sums, fp32 queries
    static constexpr int kRun = 1024 / NJ;  // and half precision
    // unit u of token row r sits at u ^ swz(r): the fragment loads are then
    // free of bank conflicts (8 rows x 16 bytes, or 4 rows 2 apart)
    static __device__ __forceinline__ int swz(int r) { return (r >> (U == 8 ? 0 : U == 4 ? 1 : 2)) & (U - 1); }
};

struct Q4Split {
    float* scratch;    // parts: [2 * warps][heads][HD], then their maxima and sums [2 * warps][heads][2]
    int4* joins;       // per unit, or per warp where the units are more: {unit, first part, its warp, last warp or -1}
    int by_unit;
    int heads;         // query heads of a unit at most
    int chunks;        // units per kv head
    uint32_t page_mul; // t / page = (2 t page_mul >> 32) >> page_shift for t < 2^31
    int page_shift;
    int cluster;       // CTAs to a unit (0: runs over all units)
};

// Stages of a query row's context, per unit.
template <int HD>
__device__ __forceinline__ int q4_stages(const AttnQ4Args& a, int64_t row) {
    const int ctx = max(0, min(a.ctx_len[row], (int)a.max_ctx));
    return (ctx + Q4Tile<HD>::TT - 1) / Q4Tile<HD>::TT;
}

// A place in the row of stages.
struct Q4Place {
    int row, kvh, chunk;
    int stage, stages;  // of this unit
};

// words b = 0 .. NB - 1 at 32-bit word t * NB + b of a swizzled row
template <int HD>
__device__ __forceinline__ void load_words(uint32_t (&w)[HD / 32], const uint8_t* tile, int row, int t) {
    using X = Q4Tile<HD>;
    const uint8_t* r = tile + row * (HD / 2);
    if constexpr (HD == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(r + (((t >> 1) ^ X::swz(row)) * 16 + (t & 1) * 8));
        w[0] = v.x, w[1] = v.y;
    } else if constexpr (HD == 128) {
        const uint4 v = *reinterpret_cast<const uint4*>(r + (t ^ X::swz(row)) * 16);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(r + ((2 * t) ^ X::swz(row)) * 16);
        const uint4 u = *reinterpret_cast<const uint4*>(r + ((2 * t + 1) ^ X::swz(row)) * 16);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w, w[4] = u.x, w[5] = u.y, w[6] = u.z, w[7] = u.w;
    }
}
// bf16 scales of tokens row, row + 1 (row even), packed pairs of blocks: s[0 .. NB/2) of row, the rest of row + 1
template <int HD>
__device__ __forceinline__ void load_scales(uint32_t (&s)[HD / 32], const uint8_t* scales, int row) {
    const uint8_t* p = scales + row * (HD / 16);
    if constexpr (HD == 64) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        s[0] = v.x, s[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < HD / 128; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
            s[4 * i] = v.x, s[4 * i + 1] = v.y, s[4 * i + 2] = v.z, s[4 * i + 3] = v.w;
        }
    }
}
// scale of block b (compile time) of the first (k = 0) or second token
template <int HD>
__device__ __forceinline__ float scale_of(const uint32_t (&s)[HD / 32], int k, int b) {
    const uint32_t w = s[k * (HD / 64) + b / 2];
    return __uint_as_float(b % 2 ? w & 0xffff0000u : w << 16);
}

// A 32-bit address of this CTA's shared memory as the same place of CTA `rank`
// of the cluster, and a load from there.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t smem, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// CL: a cluster of sp.cluster CTAs for each unit instead, its warps sharing the
// unit's stages; the parts stay in shared memory, where the cluster joins them.
template <class T, int HD, bool PACK, bool CL>
__global__ void __launch_bounds__(kWarps * 32, HD <= 128 ? 3 : 2) attn_q4_decode_kernel(AttnQ4Args a, Q4Split sp) {
    using X = Q4Tile<HD>;
    constexpr int TT = X::TT, NB = X::NB, NJ = X::NJ;
    constexpr bool kTwo = sizeof(T) == 4;  // two fp16 parts
    static_assert(!PACK || kTwo, "packing is for two parts");
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int G = (int)(a.n_head / a.n_head_kv), H = (int)a.n_head_kv, upr = H * sp.chunks;

    const int n_row = (int)a.n_q;
    uint32_t s0, base, longer, wid;
    int count;
    Q4Place at{0, 0, 0, 0, 1};
    if constexpr (CL) {
        // ---- this warp's stages of the cluster's unit; warp numbers run over the
        // CTAs first
        const int unit = (int)(blockIdx.x / (unsigned)sp.cluster);
        at.row = unit / upr;
        at.kvh = unit % upr / sp.chunks;
        at.chunk = unit % sp.chunks;
        at.stages = seq_of_row(a, at.row) < 0 ? 0 : q4_stages<HD>(a, at.row);
        const uint32_t W = (uint32_t)sp.cluster * kWarps;
        wid = (uint32_t)warp * sp.cluster + cluster_rank();
        base = (uint32_t)at.stages / W, longer = (uint32_t)at.stages - base * W;
        s0 = wid * base + min(wid, longer);
        count = (int)(base + (wid < longer));
        at.stage = (int)s0;
    } else {
        pdl_trigger();  // the join may be set up as soon as there is room
        // ---- this warp's run of stages.  Thread i sums the stages of rows i R ..
        // i R + R - 1; the warp finds the thread, then the row, where its run starts.
        // (The host sees to it that all of this fits 32 bits.)
        const int R = (n_row + kWarps * 32 - 1) / (kWarps * 32);
        int* before = reinterpret_cast<int*>(smem);  // [129 + 4], in the ring's place
        int upto = 0;
        for (int i = 0, r = threadIdx.x * R; i < R && r < n_row; ++i, ++r) upto += q4_stages<HD>(a, r);
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, k);
            if (lane >= k) upto += x;
        }
        if (lane == 31) before[kWarps * 32 + 1 + warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += before[kWarps * 32 + 1 + w];
        before[threadIdx.x + 1] = upto;
        if (threadIdx.x == 0) before[0] = 0;
        __syncthreads();
        const uint32_t total = (uint32_t)before[kWarps * 32] * (uint32_t)upr;
        // `longer` warps take base + 1 stages, the others base.  Warp numbers run
        // over the CTAs first, so that few stages spread over all SMs.
        const uint32_t W = min(gridDim.x * kWarps, total);
        wid = (uint32_t)warp * gridDim.x + blockIdx.x;
        base = W ? total / W : 0, longer = total - base * W;
        s0 = wid * base + min(wid, longer);
        count = wid < W ? (int)(base + (wid < longer)) : 0;
        if (count) {
            int n = 0;
#pragma unroll
            for (int k = 0; k < kWarps; ++k)
                n += __popc(__ballot_sync(0xffffffffu, (uint32_t)before[k * 32 + lane] * (uint32_t)upr <= s0));
            uint32_t rest = s0 - (uint32_t)before[n - 1] * (uint32_t)upr;
            at.row = (n - 1) * R;
            while (true) {
                at.stages = q4_stages<HD>(a, at.row);
                if (rest < (uint32_t)at.stages * (uint32_t)upr) break;
                rest -= (uint32_t)at.stages * (uint32_t)upr;
                ++at.row;
            }
            const uint32_t u = rest / (uint32_t)at.stages;
            at.stage = (int)(rest - u * (uint32_t)at.stages);
            at.kvh = (int)(u / (uint32_t)sp.chunks);
            at.chunk = (int)(u % (uint32_t)sp.chunks);
        }
        __syncthreads();  // `before` has been read
        // rows with no tokens give zeros, and nothing to join
        for (int r = blockIdx.x; r < n_row; r += gridDim.x)
            if (min(a.ctx_len[r], (int)a.max_ctx) <= 0) {
                for (int i = threadIdx.x; i < (int)a.n_head * HD; i += kWarps * 32)
                    static_cast<T*>(a.out)[r * (int64_t)a.out_stride + i] = from_f32<T>(0.0f);
                for (int i = threadIdx.x; sp.by_unit && i < upr; i += kWarps * 32)
                    sp.joins[(int64_t)r * upr + i].w = -1;
            }
        if (!sp.by_unit && lane == 0) sp.joins[wid].w = -1;
        if (!count) return;
    }
    auto next_unit = [&](Q4Place& p) {
        if (CL) return;
        p.stage = 0;
        if (++p.chunk < sp.chunks) return;
        p.chunk = 0;
        if (++p.kvh < H) return;
        p.kvh = 0;
        do {
            if (++p.row >= n_row) return;
            p.stages = q4_stages<HD>(a, p.row);
        } while (p.stages == 0);
    };

    uint8_t* ring = smem + warp * X::kRing;

    // ---- copies.  Lane l looks the cache slots of tokens l (and l + 32) of a
    // stage up, one stage ahead of its copies; `exists` has a bit for each that
    // is there.
    constexpr int LT = TT > 32 ? TT / 32 : 1;
    uint32_t slots[LT], exists;
    Q4Place ahead = at;
    int left = count;       // stages to copy
    const int32_t* table;   // of the sequence being copied
    int ctx;
    uint32_t head_slot;
    const uint32_t page = (uint32_t)a.page, page_rows = (uint32_t)H * page;
    auto new_unit = [&] {
        const int seq = seq_of_row(a, ahead.row);
        table = a.block_table + (int64_t)max(seq, 0) * (int64_t)a.max_pages;
        ctx = seq < 0 ? 0 : max(0, min(a.ctx_len[ahead.row], (int)a.max_ctx));
        head_slot = (uint32_t)ahead.kvh * page;
    };
    auto look_up = [&] {
        exists = 0;
#pragma unroll
        for (int i = 0; i < LT; ++i) {
            const uint32_t tok = (uint32_t)ahead.stage * TT + lane + 32 * i;
            slots[i] = 0;
            if (tok < (uint32_t)ctx && (TT >= 32 || lane < TT)) {
                const uint32_t pi = __umulhi(tok << 1, sp.page_mul) >> sp.page_shift;
                const uint32_t pg = (uint32_t)table[pi];
                if (pg < (uint32_t)a.n_pages) {
                    slots[i] = pg * page_rows + (head_slot + tok - pi * page);
                    exists |= 1u << i;
                }
            }
        }
    };
    // a missing token's nibbles are those of slot 0 -- its scales are zeros and
    // its score -inf -- so only the scale copies carry a size
    const uint8_t* k_unit = a.k_pages + lane % X::U * 16;
    const uint8_t* v_unit = a.v_pages + lane % X::U * 16;
    uint32_t valid[kStages][LT];  // tokens that are there: [0] of the stage computed next
    auto issue = [&](uint32_t st, int k) {
#pragma unroll
        for (int i = 0; i < 2048 / 16 / 32; ++i) {
            const int r = (i * 32 + lane) / X::U;  // unit lane % U of token r
            const uint32_t sl = __shfl_sync(0xffffffffu, slots[LT == 1 ? 0 : i * (32 / X::U) / 32], r & 31);
            const uint32_t dst = st + r * (HD / 2) + ((lane % X::U ^ X::swz(r)) * 16);
            cp_async16(dst, k_unit + (uint64_t)sl * (HD / 2));
            cp_async16(dst + 2048, v_unit + (uint64_t)sl * (HD / 2));
        }
#pragma unroll
        for (int i = 0; i < LT; ++i) {
            const bool ok = exists >> i & 1u;
            if (TT >= 32 || lane < TT) {
                const uint64_t off = (uint64_t)slots[i] * NB;
                const uint32_t dst = st + 4096 + (lane + 32 * i) * (NB * 2);
                cp_async_fill<NB * 2>(dst, a.k_scales + off, ok ? NB * 2 : 0);
                cp_async_fill<NB * 2>(dst + X::kScale, a.v_scales + off, ok ? NB * 2 : 0);
            }
            valid[k][i] = __ballot_sync(0xffffffffu, ok);
        }
    };
    const uint32_t ring_s = smem_u32(ring);
    new_unit();
    look_up();
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) {
        if (left > 0) {
            issue(ring_s + k * X::kBytes, k);
            if (--left) {
                if (++ahead.stage == ahead.stages) next_unit(ahead), new_unit();
                look_up();
            }
        }
        cp_async_commit();
    }

    // ---- the queries as A fragments.  Row g of the fragment is query head
    // hrow; k slots 2t, 2t + 1, 2t + 8, 2t + 9 of step s of block b are
    // dimensions 32 b + 8 t + {0, 4, 1, 5} + 2 s, the last two divided by 16.
    const int hrow = PACK ? (g & 3) : g;
    uint32_t qa[NB][2][kTwo ? 4 : 2];
    float c_h;

    const uint64_t bias0 = held_pair(-8388616.0f, -8388736.0f), bias1 = held_pair(-8390656.0f, -8421376.0f);
    const uint32_t first = g >= 4 ? 0xffffe000u : 0u;
    float o[NB][2][4];  // [block][dims 4g + 2 mu + {0, 1}][heads 2t, 2t + 1 of rows g, g + 8]
    // The tensor core cuts its running sums instead of rounding them (2e-8 to 4e-8 of
    // the sum an MMA).  fp32 queries: every 32 MMAs, and whenever the reference
    // moves, the outputs are added, rounded, to totals in shared memory and start
    // from zero.  131,071 tokens: relative error 1.6e-6 to 2.3e-6 without, 4.5e-7 to
    // 8.8e-7 so (every 16: 3.6e-7 to 5.0e-7), for 59.5 us instead of 56.0.
    // Half precision: every 1,024 MMAs, outside the loop over the stages (inside it, as
    // above, 64 x 2,000 tokens of 8 kv heads took 80 us for 58: registers).  Outputs of
    // values of one sign after 262,144 tokens in one warp: 1.1e-3 short without, four
    // times fp16's rounding, 2.7e-5 so.
    float4* total = reinterpret_cast<float4*>(smem + kWarps * X::kRing + warp * X::kTotal) + lane;
    float* total_m = reinterpret_cast<float*>(total - lane + HD * 2) + lane;
    bool held = false;  // something is in the totals
    float m_run = -INFINITY, l_run = 0.0f;
    auto add_total = [&] {  // to the outputs, on their reference (fp32 queries' totals are always on it)
        if ((CL && !kTwo) || !held) return;
        uint64_t aa = 0;
        if constexpr (!kTwo) {
            const float alpha = m_run == -INFINITY ? 0.0f : ex2(*total_m - m_run);
            aa = pair(__shfl_sync(0xffffffffu, alpha, 8 * t), __shfl_sync(0xffffffffu, alpha, 8 * t + 4));
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float(&x)[4] = o[b][m];
                const float4 y = total[(2 * b + m) * 32];
                if constexpr (kTwo) {
                    x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
                } else {
                    unpair(tc::f2_fma(pair(y.x, y.y), aa, pair(x[0], x[1])), x[0], x[1]);
                    unpair(tc::f2_fma(pair(y.z, y.w), aa, pair(x[2], x[3])), x[2], x[3]);
                }
            }
    };
    uint32_t off = 0, refill = (kStages - 1) * X::kBytes;  // of the stage computed, and of the one copied into
    if (CL && !count && lane < sp.heads)  // nothing of this warp's counts
        *reinterpret_cast<float2*>(ring + sp.heads * HD * 4 + lane * 8) = make_float2(-INFINITY, 0.0f);
    for (int n = 0; n < count;) {
        // this warp's part of the unit: stages at.stage .. end - 1
        const int from = at.stage, end = min(at.stages, from + count - n), start = n;
        const int h0 = at.kvh * G + at.chunk * sp.heads, nh = min(sp.heads, G - at.chunk * sp.heads);
        const T* q = static_cast<const T*>(a.q) + (int64_t)at.row * (int64_t)a.q_stride +
                     (int64_t)(h0 + min(hrow, nh - 1)) * HD;
        float x[NB][8], mx = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            load_n<8, true>(q + 32 * b + 8 * t, x[b]);
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[b][i]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // times 2^e: the largest below 2^15, whatever its size (e > 100 would take the
        // scores' factor out of range, and queries that small need no more bits)
        const int e = min(100, 14 - ((int)(__float_as_uint(mx) >> 23) - 127));
        const float up = pow2i(e);
        c_h = fmaxf(a.scale * 1.44269504088896341f * pow2i(-e), 1e-37f);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[b][i] *= up;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const float f[4] = {x[b][2 * s], x[b][2 * s + 4], x[b][2 * s + 1] * 0.0625f,
                                    x[b][2 * s + 5] * 0.0625f};
                float lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) lo[i] = f[i] - __half2float(__float2half_rn(f[i]));
                if constexpr (kTwo) {
                    qa[b][s][0] = pack_half2(f[0], f[1]);
                    qa[b][s][1] = pack_half2(lo[0], lo[1]);
                    qa[b][s][2] = pack_half2(f[2], f[3]);
                    qa[b][s][3] = pack_half2(lo[2], lo[3]);
                } else {
                    qa[b][s][0] = pack_half2(f[0], f[1]);
                    qa[b][s][1] = pack_half2(f[2], f[3]);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b][m][i] = 0.0f;
        m_run = -INFINITY;
        l_run = 0.0f;
        held = false;
        for (int stop = kTwo || CL ? end : min(end, from + X::kRun);; stop = min(end, stop + X::kRun)) {
            for (; at.stage < stop; ++at.stage, ++n) {
                cp_async_wait<kStages - 2>();
                __syncwarp();
                const uint8_t* kt = ring + off;
                const uint8_t* vt = kt + 2048;
                const uint8_t* ksc = kt + 4096;
                const uint8_t* vsc = ksc + X::kScale;

                // ---- scores
                float sc[NJ][2];
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    uint32_t w[NB], d[NB];
                    load_words<HD>(w, kt, 8 * j + g, t);
                    load_scales<HD>(d, ksc, 8 * j + 2 * t);
                    uint64_t sum = 0;  // two zeros
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t x = k ? w[b] >> 8 : w[b];
                            uint32_t qf[4];
                            if constexpr (kTwo) {
                                qf[0] = qa[b][k][0], qf[1] = qa[b][k][1], qf[2] = qa[b][k][2], qf[3] = qa[b][k][3];
                            } else {
                                qf[0] = qa[b][k][0], qf[1] = 0, qf[2] = qa[b][k][1], qf[3] = 0;
                            }
                            mma16816(c, qf, nib_lo(x), nib_hi(x), c);
                        }
                        const uint64_t dd = pair(scale_of<HD>(d, 0, b), scale_of<HD>(d, 1, b));
                        uint64_t cc = pair(c[0], c[1]);
                        if constexpr (kTwo) cc = f2_add(cc, pair(c[2], c[3]));
                        sum = tc::f2_fma(cc, dd, sum);
                    }
                    unpair(sum, sc[j][0], sc[j][1]);
                }
                // tokens that do not exist
#pragma unroll
                for (int i = 0; i < LT; ++i) {
                    const uint32_t v = valid[0][i], full = TT >= 32 ? 0xffffffffu : (1u << (TT & 31)) - 1u;
                    if (v != full) {
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
                            if (j / 4 == i) {
                                const uint32_t k = v >> (8 * (j % 4) + 2 * t);
                                if (!(k & 1u)) sc[j][0] = -INFINITY;
                                if (!(k & 2u)) sc[j][1] = -INFINITY;
                            }
                    }
                }
                // ---- running maximum, weights
                float mx = sc[0][0];
#pragma unroll
                for (int j = 0; j < NJ; ++j) mx = fmaxf(mx, fmaxf(sc[j][0], sc[j][1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                // The reference m follows the maximum only once that is 2^8 above it:
                // weights up to 2^8 do no harm, and the outputs are seldom rescaled.
                mx *= c_h;
                const bool sum = kTwo && at.stage != from && (at.stage - from) % X::kFlush == 0;
                if (sum || __any_sync(0xffffffffu, mx > m_run + 8.0f)) {
                    const float m_new = fmaxf(m_run, mx), alpha = m_new == -INFINITY ? 0.0f : ex2(m_run - m_new);
                    l_run *= alpha;
                    const uint64_t aa =
                    pair(__shfl_sync(0xffffffffu, alpha, 8 * t), __shfl_sync(0xffffffffu, alpha, 8 * t + 4));
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            float(&x)[4] = o[b][m];
                            if (kTwo && at.stage == from) continue;  // zeros
                            uint64_t u = pair(x[0], x[1]), v = pair(x[2], x[3]);
                            if constexpr (kTwo) {
                                if (held) {
                                    const float4 y = total[(2 * b + m) * 32];
                                    u = f2_add(u, pair(y.x, y.y)), v = f2_add(v, pair(y.z, y.w));
                                }
                            }
                            unpair(tc::f2_mul(u, aa), x[0], x[1]);
                            unpair(tc::f2_mul(v, aa), x[2], x[3]);
                            if constexpr (kTwo) {
                                total[(2 * b + m) * 32] = make_float4(x[0], x[1], x[2], x[3]);
                                x[0] = x[1] = x[2] = x[3] = 0.0f;
                            }
                        }
                    if constexpr (kTwo) held = at.stage != from;
                    m_run = m_new;
                }
                const float m_use = m_run == -INFINITY ? 0.0f : m_run;
                // ---- outputs, 8 tokens at a time
                const int half = (g & 1) * 16;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float p[2];
                    uint32_t d[NB], w[2][NB];
                    load_scales<HD>(d, vsc, 8 * j + 2 * t);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        p[i] = ex2(fmaf(sc[j][i], c_h, -m_use));
                        l_run += p[i];
                        load_words<HD>(w[i], vt, 8 * j + 2 * t + i, g >> 1);
                    }
                    const uint64_t pp = pair(p[0], p[1]);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float v[2];
                        const uint64_t vv = tc::f2_mul(pp, pair(scale_of<HD>(d, 0, b), scale_of<HD>(d, 1, b)));
                        unpair(vv, v[0], v[1]);
                        if constexpr (!kTwo) v[0] = near11(v[0]), v[1] = near11(v[1]);
                        const uint32_t x0 = w[0][b] >> half, x1 = w[1][b] >> half;
                        float f0[4], f1[4];  // rows g, g + 8 of the first token, then of the second
                        values2<0>(x0, bias0, f0[0], f0[1]);
                        values2<0>(x1, bias0, f0[2], f0[3]);
                        values2<2>(x0, bias1, f1[0], f1[1]);
                        values2<2>(x1, bias1, f1[2], f1[3]);
                        if constexpr (PACK) {
                            // columns 0..3: v, cut to 11 bits by the MMA; 4..7: v less its first 11 bits
                            const uint64_t cut = pair(-__uint_as_float(__float_as_uint(v[0]) & first),
                                                      -__uint_as_float(__float_as_uint(v[1]) & first));
                            unpair(f2_add(vv, cut), v[0], v[1]);
                        }
                        mma1688(o[b][0], f0, v[0], v[1]);
                        mma1688(o[b][1], f1, v[0], v[1]);
                        if constexpr (kTwo && !PACK) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) v[i] -= __uint_as_float(__float_as_uint(v[i]) & 0xffffe000u);
                            mma1688(o[b][0], f0, v[0], v[1]);
                            mma1688(o[b][1], f1, v[0], v[1]);
                        }
                    }
                }
                // ---- the next copies, into the stage used before this one
                __syncwarp();
#pragma unroll
                for (int k = 0; k + 1 < kStages; ++k)
#pragma unroll
                    for (int i = 0; i < LT; ++i) valid[k][i] = valid[k + 1][i];
                if (left > 0) {
                    issue(ring_s + refill, kStages - 2);
                    if (--left) {
                        if (++ahead.stage == ahead.stages) next_unit(ahead), new_unit();
                        look_up();
                    }
                }
                cp_async_commit();
                refill = off;
                off = off + X::kBytes == X::kRing ? 0 : off + X::kBytes;
            }
            if (kTwo || CL || stop == end) break;
            add_total();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    total[(2 * b + m) * 32] = make_float4(o[b][m][0], o[b][m][1], o[b][m][2], o[b][m][3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[b][m][i] = 0.0f;
                }
            *total_m = m_run;
            held = true;
        }

        // ---- the unit's end, or the run's
        add_total();
        const bool done = at.stage == at.stages;
        const bool whole = !CL && done && from == 0;
        float l = l_run + __shfl_xor_sync(0xffffffffu, l_run, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int64_t part = 2 * (int64_t)wid + (start == 0 ? 0 : 1);
        float* dst = CL ? reinterpret_cast<float*>(ring) : whole ? nullptr : sp.scratch + part * sp.heads * HD;
        float* ml = CL ? dst + sp.heads * HD
                       : sp.scratch + ((int64_t)gridDim.x * kWarps * 2 * HD + part * 2) * sp.heads;
        if constexpr (CL) {  // the ring is free once its last copies have come
            cp_async_wait<0>();
            __syncwarp();
        }
        T* out = static_cast<T*>(a.out) + (int64_t)at.row * (int64_t)a.out_stride + (int64_t)h0 * HD;
        if (!whole && t == 0 && g < nh)
            *reinterpret_cast<float2*>(ml + 2 * g) = make_float2(m_run, l);
        // sums of the two heads of this lane's columns
        float inv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = __shfl_sync(0xffffffffu, l, 8 * t + 4 * i);
            inv[i] = !whole ? 1.0f : x == 0.0f ? 0.0f : 1.0f / x;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = o[b][m][i];
                    if constexpr (PACK) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);  // columns h and h + 4
                }
                const int d = 32 * b + 4 * g + 2 * m;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int h = 2 * t + i;
                    if (h >= nh) continue;
                    // rows g and g + 8: nibbles 2 m and 2 m + 1
                    const float y0 = v[i] * (m ? 1.0f / 256 : 1.0f), y1 = v[2 + i] * (m ? 1.0f / 4096 : 1.0f / 16);
                    if (whole) {
                        out[h * HD + d] = from_f32<T>(y0 * inv[i]);
                        out[h * HD + d + 1] = from_f32<T>(y1 * inv[i]);
                    } else {
                        *reinterpret_cast<float2*>(dst + h * HD + d) = make_float2(y0, y1);
                    }
                }
            }
        if (!CL && done && lane == 0 && (sp.by_unit || !whole)) {
            const int64_t unit = ((int64_t)at.row * H + at.kvh) * sp.chunks + at.chunk;
            int4 j = make_int4((int)unit, 0, 0, -1);
            if (!whole) {  // the unit's first stage, and the warp that had it
                const uint32_t u0 = s0 + (uint32_t)start - (uint32_t)from, edge = longer * (base + 1);
                const uint32_t w0 = u0 < edge ? u0 / (base + 1) : longer + (u0 - edge) / base;
                const bool at_start = u0 == w0 * base + min(w0, longer);
                j = make_int4((int)unit, (int)(2 * w0 + (at_start ? 0 : 1)), (int)w0, (int)wid);
            }
            sp.joins[sp.by_unit ? unit : wid] = j;
        }
        if (done) next_unit(at);
    }

    if constexpr (CL) {
        // ---- the join, out = sum_w 2^(m_w - m) o_w / sum_w 2^(m_w - m) l_w: over the
        // CTA's warps, then over the cluster's CTAs, each of which takes a share of
        // the columns (4 dimensions of a head).  What a part without tokens holds
        // does not count: its sum is zero.  (Its maximum is -inf, but so is that of
        // a part whose scores are all NaN, and that one's NaN has to be seen.)
        const int h0 = at.kvh * G + at.chunk * sp.heads, nh = min(sp.heads, G - at.chunk * sp.heads);
        const int columns = nh * (HD / 4), ml_at = sp.heads * HD;  // in floats; the CTA's own after the warp's
        auto add = [](float f, const float4& x, float4& y) {
            y.x = fmaf(f, x.x, y.x), y.y = fmaf(f, x.y, y.y), y.z = fmaf(f, x.z, y.z), y.w = fmaf(f, x.w, y.w);
        };
        __syncthreads();
        for (int c = threadIdx.x; c < columns; c += kWarps * 32) {
            const int h = c / (HD / 4);
            float2 x[kWarps];
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                x[w] = reinterpret_cast<const float2*>(smem + w * X::kRing + ml_at * 4)[h];
                m = fmaxf(m, x[w].x);
            }
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (x[w].y == 0.0f) continue;
                const float f = ex2(x[w].x - m);
                l = fmaf(f, x[w].y, l);
                add(f, reinterpret_cast<const float4*>(smem + w * X::kRing)[c], y);
            }
            reinterpret_cast<float4*>(smem)[c] = y;
            if (c % (HD / 4) == 0) reinterpret_cast<float2*>(smem + ml_at * 4 + 64)[h] = make_float2(m, l);
        }
        cluster_barrier();
        T* out = static_cast<T*>(a.out) + (int64_t)at.row * (int64_t)a.out_stride + (int64_t)h0 * HD;
        const int share = (columns + sp.cluster - 1) / sp.cluster, c1 = min(columns, share * ((int)cluster_rank() + 1));
        for (int c = share * (int)cluster_rank() + threadIdx.x; c < c1; c += kWarps * 32) {
            const uint32_t ml = smem_u32(smem) + ml_at * 4 + 64 + c / (HD / 4) * 8, col = smem_u32(smem) + c * 16;
            float2 x[8];
            float4 u[8];
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= sp.cluster) continue;
                x[r] = cluster_load2(cluster_addr(ml, r));
                u[r] = cluster_load4(cluster_addr(col, r));
            }
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < sp.cluster) m = fmaxf(m, x[r].x);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= sp.cluster || x[r].y == 0.0f) continue;
                const float f = ex2(x[r].x - m);
                l = fmaf(f, x[r].y, l);
                add(f, u[r], y);
            }
            const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int d = 0; d < 4; ++d) out[c * 4 + d] = from_f32<T>(l == 0.0f ? 0.0f : v[d] / l);
        }
        cluster_barrier();  // nobody's shared memory goes before it has been read
    }
}

// Joins the parts of one unit: out = sum_r 2^(m_r - m) o_r / sum_r 2^(m_r - m)
// l_r, a head at a time (one CTA per head where the units are few).  The parts
// are dealt to groups of HD / 4 threads, four of a group's parts in flight,
// each group with a maximum of its own; the groups are joined in shared memory.
constexpr int kJoin = 1024;
template <class T, int HD>
__global__ void __launch_bounds__(kJoin) attn_q4_join_kernel(AttnQ4Args a, Q4Split sp, int64_t warps) {
    constexpr int kLane = HD / 4, kGroups = kJoin / kLane;
    __shared__ float red[kGroups][HD + 2];
    const int G = (int)(a.n_head / a.n_head_kv), H = (int)a.n_head_kv, hs = sp.heads;
    pdl_wait();
    const int4 j = sp.joins[blockIdx.x];
    if (j.w < 0) return;
    const int chunk = j.x % sp.chunks, kvh = j.x / sp.chunks % H, parts = j.w - j.z + 1;
    const int64_t row = j.x / sp.chunks / H;
    const int nh = min(hs, G - chunk * hs);
    const float* ml = sp.scratch + 2 * warps * HD * hs;
    const int d = threadIdx.x % kLane * 4, grp = threadIdx.x / kLane, groups = blockDim.x / kLane;
    auto part = [&](int r) -> int64_t { return r == 0 ? j.y : 2 * (int64_t)(j.z + r); };
    for (int h = blockIdx.y; h < nh; h += gridDim.y) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f}, top = -INFINITY, l = 0.0f;
        for (int r = grp; r < parts; r += 4 * groups) {
            float2 x[4];
            float4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t k = part(min(r + i * groups, parts - 1)) * hs + h;
                x[i] = *reinterpret_cast<const float2*>(ml + k * 2);
                u[i] = *reinterpret_cast<const float4*>(sp.scratch + k * HD + d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r + i * groups >= parts || x[i].y == 0.0f) continue;  // (no tokens: the sum, as above)
                const float m = fmaxf(top, x[i].x), e = ex2(top - m), c = ex2(x[i].x - m);
                y[0] = fmaf(c, u[i].x, e * y[0]), y[1] = fmaf(c, u[i].y, e * y[1]);
                y[2] = fmaf(c, u[i].z, e * y[2]), y[3] = fmaf(c, u[i].w, e * y[3]);
                l = fmaf(c, x[i].y, e * l);
                top = m;
            }
        }
        __syncthreads();  // the last head's sums have been read
#pragma unroll
        for (int i = 0; i < 4; ++i) red[grp][d + i] = y[i];
        if (d == 0) red[grp][HD] = l, red[grp][HD + 1] = top;
        __syncthreads();
        T* out = static_cast<T*>(a.out) + row * (int64_t)a.out_stride + (int64_t)(kvh * G + chunk * hs + h) * HD;
        for (int i = threadIdx.x; i < HD; i += blockDim.x) {
            float v = 0.0f, den = 0.0f, m = -INFINITY;
            for (int w = 0; w < groups; ++w) m = fmaxf(m, red[w][HD + 1]);
            for (int w = 0; w < groups; ++w) {
                const float c = red[w][HD] == 0.0f ? 0.0f : ex2(red[w][HD + 1] - m);
                v = fmaf(c, red[w][i], v), den = fmaf(c, red[w][HD], den);
            }
            out[i] = from_f32<T>(den == 0.0f ? 0.0f : v / den);
        }
    }
}

// CTAs of a kernel that the current GPU holds at once.
uint64_t resident_ctas(const void* kernel, int threads, int smem) {
    int per = 0, sms = 0, dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem);
    return (uint64_t)std::max(1, per * sms);
}

// `need`: only says how much scratch the launch takes.
template <class T, int HD, bool PACK>
cudaError_t launch_decode(const AttnQ4Args& a, cudaStream_t s, uint64_t* need) {
    using X = Q4Tile<HD>;
    constexpr int kHeads = PACK ? 4 : 8;
    const int smem = kWarps * (X::kRing + X::kTotal);
    auto kernel = attn_q4_decode_kernel<T, HD, PACK, false>;
    ensure_smem_attr(kernel, smem);
    static const uint64_t slots = resident_ctas(reinterpret_cast<const void*>(kernel), kWarps * 32, smem);
    Q4Split sp{};
    const uint64_t G = a.n_head / a.n_head_kv;
    sp.heads = (int)std::min<uint64_t>(kHeads, G);
    sp.chunks = (int)((G + kHeads - 1) / kHeads);
    const uint64_t units = a.n_q * a.n_head_kv * sp.chunks;
    if (units > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    int L = 0;
    while ((1ull << L) < a.page) ++L;
    sp.page_mul = (uint32_t)(((1ull << (31 + L)) + a.page - 1) / a.page);
    sp.page_shift = L;
    const uint64_t most = units * ((a.max_ctx + X::TT - 1) / X::TT);  // stages
    if (most >= (1ull << 31) || a.n_q > 0x7fffff00ull) return cudaErrorInvalidConfiguration;  // counted in 32 bits
    // Short contexts of few units: a cluster a unit, of 8 CTAs or the fewest that give
    // a warp one stage, while the GPU holds them all at once and none has more than
    // kShort stages to a warp.  Runs over all units and a second kernel that joins
    // them, against this (fp32 queries, head_dim 128; both 3 to 6% less than with the
    // rounded totals above):
    //    768 tokens, 32 units     9.3 ->  6.1 us     4,096 tokens, 32 units  16.2 -> 11.1 us
    //    1,000 tokens, 64 units  15.1 ->  8.4 us     4,000 tokens, 64 units  23.6 -> 17.8 us
    //    250 tokens, 256 units   14.1 ->  8.4 us     1,000 tokens, 256 units 23.9 -> 17.8 us
    //    8,192 tokens, 8 units   13.5 -> 13.1 us (8 stages); 16,384: 17.7 -> 21.8 us
    // More units than fit at once: 64 ragged contexts x 32 heads 45.6 -> 53.8 us.
    const uint64_t longest = (a.max_ctx + X::TT - 1) / X::TT;
    uint64_t cluster = 8;
    while (cluster > 1 && (cluster / 2 * kWarps >= longest || units * cluster > slots)) cluster /= 2;
    if (units * cluster <= slots && longest <= cluster * kWarps * kShort) {
        if (need) {
            *need = 0;
            return cudaSuccess;
        }
        sp.cluster = (int)cluster;
        const int smem = kWarps * (X::kRing + (sizeof(T) == 4 ? X::kTotal : 0));
        auto one = attn_q4_decode_kernel<T, HD, PACK, true>;
        ensure_smem_attr(one, smem);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(units * cluster)), cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = smem, cfg.stream = s;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr, cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, one, a, sp);
    }
    const uint64_t grid = std::max<uint64_t>(1, std::min<uint64_t>(slots, most)), warps = grid * kWarps;
    sp.by_unit = units <= warps;
    const uint64_t joins = sp.by_unit ? units : warps;
    const uint64_t parts = 2 * warps * sp.heads * (HD + 2) * 4;
    if (need) {
        *need = parts + joins * sizeof(int4);
        return cudaSuccess;
    }
    uint8_t* scratch = static_cast<uint8_t*>(a.workspace);
    if (!scratch) {
        const uint64_t bytes = parts + joins * sizeof(int4);
        if (cudaError_t e = scratch_alloc(reinterpret_cast<void**>(&scratch), bytes, s)) return e;
    }
    sp.scratch = reinterpret_cast<float*>(scratch);
    sp.joins = reinterpret_cast<int4*>(scratch + parts);
    // many parts a unit: all 1024 threads; few: as many groups as there are parts, at most
    const uint64_t unit_parts = std::min(warps, most) / std::max<uint64_t>(1, std::min(units, warps)) + 2;
    const unsigned join_threads =
        (unsigned)std::min<uint64_t>(kJoin, std::max<uint64_t>(128, (unit_parts * (HD / 4) + 127) / 128 * 128));
    const dim3 join_grid((unsigned)joins, sp.by_unit ? (unsigned)sp.heads : 1u, 1u);
    kernel<<<(unsigned)grid, kWarps * 32, smem, s>>>(a, sp);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess)
        e = launch_pdl(attn_q4_join_kernel<T, HD>, join_grid, dim3(join_threads), 0, s, a, sp, (int64_t)warps);
    if (!a.workspace) cudaFreeAsync(scratch, s);
    return e;
}
template <class T>
cudaError_t attn_decode(const AttnQ4Args& a, cudaStream_t s, uint64_t* need) {
    if constexpr (sizeof(T) == 4) {
        if (a.n_head / a.n_head_kv <= 4) {
            if (a.hd == 64) return launch_decode<T, 64, true>(a, s, need);
            if (a.hd == 128) return launch_decode<T, 128, true>(a, s, need);
            return launch_decode<T, 256, true>(a, s, need);
        }
    }
    if (a.hd == 64) return launch_decode<T, 64, false>(a, s, need);
    if (a.hd == 128) return launch_decode<T, 128, false>(a, s, need);
    return launch_decode<T, 256, false>(a, s, need);
}
cudaError_t decode_of(int type, const AttnQ4Args& a, cudaStream_t s, uint64_t* need) {
    if (type == kTypeF32) return attn_decode<float>(a, s, need);
    if (type == kTypeF16) return attn_decode<__half>(a, s, need);
    return attn_decode<__nv_bfloat16>(a, s, need);
}

// Chunks go row by row through the kernel above while they are small: a row and
// kv head costs it 46 to 57 ps a token (head_dim 128, fp32), whereas a wave of the
// tensor-core kernel's CTAs takes 25 ns a token however few of its 128 rows are
// used -- as much as 550 rows.  Measured by head_dim 64, 128, 256: 820, 550, 770 rows
// (fp32 queries; 700, 490, 700 for groups above 4), 640, 425, 450 (half precision).
// The bounds are set low, since a causal chunk's first rows are cheap row by row and
// its tiles are not.
// Only the tiles that hold rows count, each sequence's last one part empty; a CTA
// without rows leaves its SM after 1.1 us, a wave's 25 ns for 44 tokens.  One chunk of
// 2,048 rows and 63 single rows after 700 tokens, 32 heads x 128: fp32 775 us (row by
// row 5,085), 32 heads / 8 bf16 290 us (1,259).
bool rows_one_by_one(int type, const AttnQ4Args& a) {
    const uint64_t G = a.n_head / a.n_head_kv, heads = type == kTypeF32 && G <= 4 ? 4 : 8;
    const uint64_t rpt = 128 / std::min<uint64_t>(G, 128), units = a.n_head_kv * ((G + 127) / 128);
    const uint64_t ctas = prefill_tiles(a, rpt) * units, grid = a.n_seq * ((a.max_q + rpt - 1) / rpt) * units;
    const uint64_t wave = type == kTypeF32 ? 520 : 350, empty = (grid - ctas) / 148;
    return a.n_q * a.n_head_kv * ((G + heads - 1) / heads) <
           wave * ((ctas + 147) / 148) + wave * 44 * empty / std::max<uint64_t>(44, a.max_ctx);
}

}  // namespace

uint64_t attn_q4_workspace(int type, const AttnQ4Args& a) {
    uint64_t need = 0;
    decode_of(type, a, nullptr, &need);
    return need;
}

cudaError_t attn_q4(int type, const AttnQ4Args& a, cudaStream_t s) {
    if (!a.n_q || !a.n_head) return cudaSuccess;
    if ((a.q_start || a.one_seq) && !rows_one_by_one(type, a)) return attn_q4_prefill(type, a, s);
    return decode_of(type, a, s, nullptr);
}

}  // namespace mvb
