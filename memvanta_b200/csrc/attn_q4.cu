// attn_q4.cu -- attention over the 4-bit paged cache (kv_q4.cuh).
//
//   out[r][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[r][h].k_t - m)
// over the first ctx_len[r] cached tokens of the row's sequence, in one pass
// with the running maximum m and sum.  A row with no tokens gives zeros; what
// lies past ctx_len, or on a page that does not exist, is never used.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.cuh"
#include "kv_q4.cuh"
#include "tc.cuh"

namespace mvb {

namespace cg = cooperative_groups;

namespace {

// The sequence of query row r (q_start ascending), by bisection.
__device__ __forceinline__ int seq_of_row(const AttnQ4Args& a, int64_t r) {
    if (!a.q_start) return (int)r;
    int lo = 0, hi = (int)a.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.q_start[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One (row, head) per CTA: four warps take every fourth token, lane l holds
// dimensions (HD / 32) l .. of the running output.
template <class T, int HD>
__global__ void __launch_bounds__(128) attn_q4_row_kernel(AttnQ4Args a) {
    constexpr int E = HD / 32;
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, kvh = h / (int)(a.n_head / a.n_head_kv), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = seq_of_row(a, r);
    const int64_t ctx = min((int64_t)a.ctx_len[r], (int64_t)min(a.max_ctx, a.max_pages * a.page));
    const T* q = static_cast<const T*>(a.q) + r * (int64_t)a.q_stride + h * HD;
    float qv[E], o[E], m = -INFINITY, sum = 0.0f;
    const int d0 = lane * E, b = d0 / 32;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        qv[i] = to_f32(q[d0 + i]) * a.scale;
        o[i] = 0.0f;
    }
    for (int64_t t = warp; t < ctx; t += 4) {
        const int64_t pg = a.block_table[(int64_t)s * (int64_t)a.max_pages + t / (int64_t)a.page];
        if (pg < 0 || pg >= (int64_t)a.n_pages) continue;
        const int64_t tok = (pg * (int64_t)a.n_head_kv + kvh) * (int64_t)a.page + t % (int64_t)a.page;
        const uint8_t* kp = a.k_pages + tok * (HD / 2);
        const uint8_t* vp = a.v_pages + tok * (HD / 2);
        float kd = bf16_bits_to_f32(a.k_scales[tok * (HD / 32) + b]), vd = bf16_bits_to_f32(a.v_scales[tok * (HD / 32) + b]);
        float dot = 0.0f, v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int d = d0 + i, at = (d % 32 / 8 * (HD / 32) + b) * 4 + d % 8 / 2, sh = d % 2 * 4;
            dot = fmaf(qv[i], (float)((int)((kp[at] >> sh) & 15) - 8) * kd, dot);
            v[i] = (float)((int)((vp[at] >> sh) & 15) - 8) * vd;
        }
        dot = warp_sum(dot);
        const float mn = fmaxf(m, dot), c = m > -INFINITY ? expf(m - mn) : 0.0f, p = expf(dot - mn);
        sum = sum * c + p;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf(p, v[i], o[i] * c);
        m = mn;
    }
    __shared__ float sm[4], ss[4], so[4][HD];
#pragma unroll
    for (int i = 0; i < E; ++i) so[warp][d0 + i] = o[i];
    if (lane == 0) sm[warp] = m, ss[warp] = sum;
    __syncthreads();
    const float mt = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float w[4], den = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = sm[i] > -INFINITY ? expf(sm[i] - mt) : 0.0f;
        den += ss[i] * w[i];
    }
    T* out = static_cast<T*>(a.out) + r * (int64_t)a.out_stride + h * HD;
    for (int d = threadIdx.x; d < HD; d += 128) {
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) y = fmaf(w[i], so[i][d], y);
        out[d] = from_f32<T>(den == 0.0f ? 0.0f : y / den);
    }
}

template <class T>
cudaError_t attn_rows(const AttnQ4Args& a, cudaStream_t s) {
    const dim3 grid((unsigned)a.n_q, (unsigned)a.n_head);
    if (a.hd == 64) attn_q4_row_kernel<T, 64><<<grid, 128, 0, s>>>(a);
    else if (a.hd == 128) attn_q4_row_kernel<T, 128><<<grid, 128, 0, s>>>(a);
    else attn_q4_row_kernel<T, 256><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
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
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(h);
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// D (16 x 8, fp32) += A (16 x 8, tf32) B (8 x 8, tf32)
__device__ __forceinline__ void mma1688(float (&d)[4], const float (&a)[4], float b0, float b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
          "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// Nibbles 0 and 4 (lo), or 1 and 5 (hi), of x as two fp16 numbers n - 8: ORed
// into 1024 they are 1024 + n, or 1024 + 16 n, and one fp16 operation is exact.
// (As fp16 subnormals n 2^-24, without that operation, the tensor core aligned
// its sum to their exponent field, 2^-14, and scores lost 4 bits.)
__device__ __forceinline__ uint32_t nib_lo(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    const __half2 h = __hadd2(reinterpret_cast<const __half2&>(r), __float2half2_rn(-1032.0f));
    return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint32_t nib_hi(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    const __half2 h = __hfma2(reinterpret_cast<const __half2&>(r), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f));
    return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
// Nibbles I, I + 1 of a token's word times its scale (twice in d): (n - 8) d in
// fp32, exact (at most 11 bits).  A nibble is masked in place and ORed into
// the mantissa of 2^23, giving 2^23 + n 2^(4 I); a packed FMA scales that back
// and takes 2^(23 - 4 I) + 8 off.  The pair are neighbours in the MMA's A
// registers (rows g, g + 8): pairs over two tokens cost a move each.
template <int I>
__device__ __forceinline__ void values2(uint32_t x, uint64_t d, float& v0, float& v1) {
    uint32_t u0, u1;
    asm("lop3.b32 %0, %1, %2, 0x4b000000, 0xea;" : "=r"(u0) : "r"(x), "n"(0xf << (4 * I)));
    asm("lop3.b32 %0, %1, %2, 0x4b000000, 0xea;" : "=r"(u1) : "r"(x), "n"(0xf0 << (4 * I)));
    constexpr float m = 1.0f / (1 << (4 * I)), k = 8388608.0f * m;
    const uint64_t n = tc::f2_fma(pair(__uint_as_float(u0), __uint_as_float(u1)), pair(m, m / 16),
                                  pair(-k - 8.0f, -k / 16 - 8.0f));
    unpair(tc::f2_mul(n, d), v0, v1);
}
__device__ __forceinline__ float to_tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return __uint_as_float(r);
}

// ---------------------------------------------------------- one query row
// A CTA of 4 warps takes one (sequence, kv head, up to 8 of its query heads)
// and a range of tokens; each warp its own 4096 / HD tokens of every fourth
// part of the range ("a stage"), through a ring of its own in shared memory
// (cp.async; no barrier between warps until the end).
//
// Both products run on the tensor cores, the cache as integers:
//  scores  (heads x tokens, m16n8k16 fp16): A = the queries, B = keys n - 8,
//          exact; each 32-block's sum is multiplied by its scale afterwards, in
//          fp32.
//  outputs (dims x heads, m16n8k8 tf32): A = the values (n - 8) d, exact in
//          tf32's 11 bits, B = the weights.  tf32 keeps their whole exponent
//          range: in fp16 a dimension whose heavy tokens are all zero lost the
//          light ones.
// fp32 queries and their weights go in as two parts of 11 bits: the queries'
// second parts are rows 8..15 of A, the weights' are columns 4..7 for up to
// four heads (PACK: rows 4..7 repeat heads 0..3, so a lane's weights are
// already there) and a second MMA for more.
constexpr int kWarps = 4, kStages = 3, kMaxSplits = 512;

template <int HD>
struct Q4Tile {
    static constexpr int TT = 4096 / HD;  // tokens of a stage: 2 KB of keys, 2 KB of values
    static constexpr int NB = HD / 32;    // scale blocks
    static constexpr int U = HD / 32;     // 16-byte units of a token's nibbles
    static constexpr int NJ = TT / 8;     // 8-token fragments
    static constexpr int kScale = TT * NB * 2;
    static constexpr int kBytes = 2 * 2048 + 2 * kScale;  // K, V, K scales, V scales
    static constexpr int kRing = kStages * kBytes;
    // unit u of token row r sits at u ^ swz(r): the fragment loads are then
    // free of bank conflicts (8 rows x 16 bytes, or 4 rows 2 apart)
    static __device__ __forceinline__ int swz(int r) { return (r >> (U == 8 ? 0 : U == 4 ? 1 : 2)) & (U - 1); }
};

struct Q4Split {       // how a launch cuts the tokens
    int splits;        // CTAs per unit: a cluster, or with scratch any number
    float* scratch;    // [units][splits][heads][HD + 2] or nullptr
    int heads;         // query heads of a unit at most
    int chunks;        // query-head chunks of 8 (4 with PACK) per kv head
    uint32_t page_mul; // t / page = t * page_mul >> page_shift for t < 2^31
    int page_shift;
};

// Tokens of each part of a context: equal, in whole CTA stages, so a short
// context takes fewer parts than there are.
__device__ __forceinline__ int q4_part(int ctx, int splits, int stage) {
    return ((ctx + splits - 1) / splits + stage - 1) / stage * stage;
}

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

template <class T, int HD, bool PACK>
__global__ void __launch_bounds__(kWarps * 32) attn_q4_decode_kernel(AttnQ4Args a, Q4Split sp) {
    using X = Q4Tile<HD>;
    constexpr int TT = X::TT, NB = X::NB, NJ = X::NJ;
    constexpr bool kTwo = sizeof(T) == 4;  // two fp16 parts
    static_assert(!PACK || kTwo, "packing is for two parts");
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int G = (int)(a.n_head / a.n_head_kv), H = (int)a.n_head_kv;
    const int split = (int)blockIdx.x % sp.splits;
    const int64_t unit = blockIdx.x / (unsigned)sp.splits;  // (row, kv head, chunk of heads)
    const int chunk = (int)(unit % sp.chunks), kvh = (int)(unit / sp.chunks % H);
    const int64_t row = unit / sp.chunks / H;
    const int h0 = kvh * G + chunk * sp.heads, nh = min(sp.heads, G - chunk * sp.heads);
    const int ctx = (int)max(0, min(a.ctx_len[row], (int)a.max_ctx));
    const int per = q4_part(ctx, sp.splits, kWarps * TT);
    const int first = (int)min((int64_t)ctx, (int64_t)split * per), last = (int)min((int64_t)ctx, (int64_t)first + per);
    if (sp.scratch && first >= last) return;

    uint8_t* ring = smem + warp * X::kRing;
    const uint32_t ring_s = smem_u32(ring);
    uint32_t* valid_ring = reinterpret_cast<uint32_t*>(smem + kWarps * X::kRing) + warp * kStages * 2;
    const int32_t* table = a.block_table + row * (int64_t)a.max_pages;

    // ---- copies.  Lane l looks the cache slots of tokens l (and l + 32) of a
    // stage up; `exists` has a bit for each that is there.
    constexpr int LT = TT > 32 ? TT / 32 : 1;
    uint32_t slots[LT], exists;
    auto look_up = [&](int base) {
        exists = 0;
#pragma unroll
        for (int i = 0; i < LT; ++i) {
            const uint32_t tok = (uint32_t)base + lane + 32 * i;
            slots[i] = 0;
            if (tok < (uint32_t)last && (TT >= 32 || lane < TT)) {
                const uint32_t pi = (uint32_t)(((uint64_t)tok * sp.page_mul) >> sp.page_shift);
                const uint32_t pg = (uint32_t)table[pi];
                if (pg < (uint32_t)a.n_pages) {
                    slots[i] = (pg * (uint32_t)H + (uint32_t)kvh) * (uint32_t)a.page + (tok - pi * (uint32_t)a.page);
                    exists |= 1u << i;
                }
            }
        }
    };
    // a missing token's nibbles are those of slot 0 -- its scales are zeros and
    // its score -inf -- so only the scale copies carry a size
    const uint8_t* k_unit = a.k_pages + lane % X::U * 16;
    const uint8_t* v_unit = a.v_pages + lane % X::U * 16;
    auto issue = [&](int s) {
        const uint32_t st = ring_s + s * X::kBytes;
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
            const uint32_t v = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) valid_ring[s * 2 + i] = v;
        }
    };
    const int base0 = first + warp * TT;
    constexpr int kStep = kWarps * TT;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (base0 + s * kStep < last) {
            look_up(base0 + s * kStep);
            issue(s);
        }
        cp_async_commit();
    }
    look_up(base0 + (kStages - 1) * kStep);

    // ---- the queries as A fragments.  Row g of the fragment is query head
    // hrow; k slots 2t, 2t + 1, 2t + 8, 2t + 9 of step s of block b are
    // dimensions 32 b + 8 t + {0, 4, 1, 5} + 2 s.
    const int hrow = PACK ? (g & 3) : g;
    uint32_t qa[NB][2][kTwo ? 4 : 2];
    float c_h;
    {
        const T* q = static_cast<const T*>(a.q) + row * (int64_t)a.q_stride + (int64_t)(h0 + min(hrow, nh - 1)) * HD;
        float x[NB][8], mx = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            load_n<8, true>(q + 32 * b + 8 * t, x[b]);
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[b][i]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // times 2^e: the largest below 2^15
        const int e = max(-100, min(100, 14 - ((int)(__float_as_uint(mx) >> 23) - 127)));
        const float up = pow2i(e);
        c_h = fmaxf(a.scale * 1.44269504088896341f * pow2i(-e), 1e-37f);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[b][i] *= up;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const float f[4] = {x[b][2 * s], x[b][2 * s + 4], x[b][2 * s + 1], x[b][2 * s + 5]};
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
    }

    float o[NB][2][4];  // [block][dims 4g + 2 mu + {0, 1}][heads 2t, 2t + 1 of rows g, g + 8]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[b][m][i] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;

    int s = 0;
    for (int base = base0; base < last; base += kStep) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        const uint8_t* kt = ring + s * X::kBytes;
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
            const uint32_t v = valid_ring[s * 2 + i], full = TT >= 32 ? 0xffffffffu : (1u << (TT & 31)) - 1u;
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
        const float m_new = fmaxf(m_run, mx * c_h), m_use = m_new == -INFINITY ? 0.0f : m_new;
        if (__any_sync(0xffffffffu, m_new != m_run)) {
            const float alpha = m_run == -INFINITY ? 0.0f : ex2(m_run - m_use);
            l_run *= alpha;
            const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    o[b][m][0] *= a0, o[b][m][1] *= a1;
                    o[b][m][2] *= a0, o[b][m][3] *= a1;
                }
            m_run = m_new;
        }
        // ---- outputs, 8 tokens at a time
        const int half = (g & 1) * 16;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float p[2], r[2];
            uint32_t d[NB], w[2][NB];
            load_scales<HD>(d, vsc, 8 * j + 2 * t);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[i] = ex2(fmaf(sc[j][i], c_h, -m_use));
                l_run += p[i];
                load_words<HD>(w[i], vt, 8 * j + 2 * t + i, g >> 1);
                if constexpr (kTwo) {
                    const float hi = __uint_as_float(__float_as_uint(p[i]) & 0xffffe000u);  // 11 bits
                    r[i] = p[i] - hi;
                    p[i] = PACK && g >= 4 ? r[i] : hi;
                } else {
                    p[i] = to_tf32(p[i]);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float dA = scale_of<HD>(d, 0, b), dB = scale_of<HD>(d, 1, b);
                const uint32_t x0 = w[0][b] >> half, x1 = w[1][b] >> half;
                float f0[4], f1[4];  // rows g, g + 8 of the first token, then of the second
                values2<0>(x0, pair(dA, dA), f0[0], f0[1]);
                values2<0>(x1, pair(dB, dB), f0[2], f0[3]);
                values2<2>(x0, pair(dA, dA), f1[0], f1[1]);
                values2<2>(x1, pair(dB, dB), f1[2], f1[3]);
                mma1688(o[b][0], f0, p[0], p[1]);
                mma1688(o[b][1], f1, p[0], p[1]);
                if constexpr (kTwo && !PACK) {
                    mma1688(o[b][0], f0, r[0], r[1]);
                    mma1688(o[b][1], f1, r[0], r[1]);
                }
            }
        }
        // ---- the next copies, into the stage used before this one
        __syncwarp();
        if (base + (kStages - 1) * kStep < last) {
            issue((s + kStages - 1) % kStages);
            look_up(base + kStages * kStep);
        }
        cp_async_commit();
        s = s + 1 == kStages ? 0 : s + 1;
    }
    pdl_trigger();  // the join may be set up
    cp_async_wait<0>();
    __syncthreads();  // the ring is reused for the warps' results

    // ---- the warps' results, then the CTA's
    float* po = reinterpret_cast<float*>(smem);      // [warp][8 heads][HD]
    float* pm = po + kWarps * 8 * HD;                // [warp][8] maxima, sums
    float* pl = pm + kWarps * 8;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (t == 0) pm[warp * 8 + g] = m_run, pl[warp * 8 + g] = l_run;
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
            if (!PACK || t < 2) {
                const int d = 32 * b + 4 * g + 2 * m;
                float* dst = po + (warp * 8 + 2 * t) * HD + d;
                *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[2]);
                *reinterpret_cast<float2*>(dst + HD) = make_float2(v[1], v[3]);
            }
        }
    __syncthreads();
    float* co = pl + kWarps * 8;     // the CTA's result [8][HD], then maxima and sums [8]
    float* cm = co + 8 * HD;
    float* cl = cm + 8;
    for (int i = threadIdx.x; i < nh * HD; i += kWarps * 32) {
        const int h = i / HD;
        float mt = -INFINITY, y = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, pm[w * 8 + h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float m = pm[w * 8 + h], c = m == -INFINITY ? 0.0f : ex2(m - mt);
            y = fmaf(c, po[w * 8 * HD + i], y);
            l = fmaf(c, pl[w * 8 + h], l);
        }
        co[i] = y;
        if (i % HD == 0) cm[h] = mt, cl[h] = l;
    }
    __syncthreads();
    T* out = static_cast<T*>(a.out) + row * (int64_t)a.out_stride + (int64_t)h0 * HD;
    if (sp.splits == 1) {
        for (int i = threadIdx.x; i < nh * HD; i += kWarps * 32) {
            const float l = cl[i / HD];
            out[i] = from_f32<T>(l == 0.0f ? 0.0f : co[i] / l);
        }
    } else if (sp.scratch) {
        float* dst = sp.scratch + (int64_t)blockIdx.x * sp.heads * (HD + 2);
        for (int i = threadIdx.x; i < nh * HD; i += kWarps * 32) dst[i] = co[i];
        if ((int)threadIdx.x < nh) {
            dst[sp.heads * HD + threadIdx.x] = cm[threadIdx.x];
            dst[sp.heads * (HD + 1) + threadIdx.x] = cl[threadIdx.x];
        }
    } else {
        // the cluster's CTAs are this unit's parts: each joins its share of the
        // elements, reading the others' results from their shared memory
        cg::cluster_group cl_grp = cg::this_cluster();
        cl_grp.sync();
        for (int i = split * (kWarps * 32) + threadIdx.x; i < nh * HD; i += sp.splits * kWarps * 32) {
            const int h = i / HD;
            float mt = -INFINITY, y = 0.0f, l = 0.0f;
            for (int r = 0; r < sp.splits; ++r) mt = fmaxf(mt, cl_grp.map_shared_rank(cm, r)[h]);
            for (int r = 0; r < sp.splits; ++r) {
                const float m = cl_grp.map_shared_rank(cm, r)[h], c = m == -INFINITY ? 0.0f : ex2(m - mt);
                y = fmaf(c, cl_grp.map_shared_rank(co, r)[i], y);
                l = fmaf(c, cl_grp.map_shared_rank(cl, r)[h], l);
            }
            out[i] = from_f32<T>(l == 0.0f ? 0.0f : y / l);
        }
        cl_grp.sync();  // nobody leaves while another reads its shared memory
    }
}

// Joins the parts of one unit's head (a CTA each): out = sum_r 2^(m_r - m) o_r
// / sum_r 2^(m_r - m) l_r, the parts dealt to groups of HD / 4 threads.
template <class T, int HD>
__global__ void __launch_bounds__(256) attn_q4_join_kernel(AttnQ4Args a, Q4Split sp) {
    constexpr int kLane = HD / 4, kGroups = 256 / kLane;
    __shared__ float c[kMaxSplits], red[kGroups][HD + 1];
    const int64_t unit = blockIdx.x;
    const int G = (int)(a.n_head / a.n_head_kv), H = (int)a.n_head_kv, hs = sp.heads, h = blockIdx.y;
    const int chunk = (int)(unit % sp.chunks), kvh = (int)(unit / sp.chunks % H);
    const int64_t row = unit / sp.chunks / H;
    if (chunk * hs + h >= G) return;
    const int ctx = (int)max(0, min(a.ctx_len[row], (int)a.max_ctx));
    const int per = q4_part(ctx, sp.splits, kWarps * Q4Tile<HD>::TT), parts = per ? (ctx + per - 1) / per : 0;
    const int64_t stride = (int64_t)hs * (HD + 2);
    const float* src = sp.scratch + unit * sp.splits * stride;
    pdl_wait();
    float mt = -INFINITY, l = 0.0f;
    for (int r = threadIdx.x; r < parts; r += 256) mt = fmaxf(mt, src[r * stride + hs * HD + h]);
    mt = warp_max(mt);
    if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = mt;
    __syncthreads();
    mt = red[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) mt = fmaxf(mt, red[0][w]);
    for (int r = threadIdx.x; r < parts; r += 256) {
        const float m = src[r * stride + hs * HD + h];
        c[r] = m == -INFINITY ? 0.0f : ex2(m - mt);
    }
    __syncthreads();
    const int d = threadIdx.x % kLane * 4, grp = threadIdx.x / kLane;
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = grp; r < parts; r += kGroups) {
        const float w = c[r];
        const float2 u = *reinterpret_cast<const float2*>(src + r * stride + h * HD + d),
                     v = *reinterpret_cast<const float2*>(src + r * stride + h * HD + d + 2);
        y[0] = fmaf(w, u.x, y[0]), y[1] = fmaf(w, u.y, y[1]);
        y[2] = fmaf(w, v.x, y[2]), y[3] = fmaf(w, v.y, y[3]);
        if (d == 0) l = fmaf(w, src[r * stride + hs * (HD + 1) + h], l);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[grp][d + i] = y[i];
    if (d == 0) red[grp][HD] = l;
    __syncthreads();
    T* out = static_cast<T*>(a.out) + row * (int64_t)a.out_stride + (int64_t)(kvh * G + chunk * hs + h) * HD;
    for (int i = threadIdx.x; i < HD; i += 256) {
        float v = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < kGroups; ++w) v += red[w][i], den += red[w][HD];
        out[i] = from_f32<T>(den == 0.0f ? 0.0f : v / den);
    }
}

template <class T, int HD, bool PACK>
cudaError_t launch_decode(const AttnQ4Args& a, cudaStream_t s) {
    using X = Q4Tile<HD>;
    constexpr int kHeads = PACK ? 4 : 8, kCta = kWarps * X::TT;
    const int merge = (kWarps * 8 * (HD + 2) + 8 * (HD + 2)) * 4;
    const int smem = std::max(kWarps * X::kRing + kWarps * kStages * 8, merge);
    auto kernel = attn_q4_decode_kernel<T, HD, PACK>;
    ensure_smem_attr(kernel, smem);
    static const int slots = [&] {  // CTAs that the GPU holds at once
        int per = 0, sms = 0, dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kWarps * 32, smem);
        return std::max(1, per * sms);
    }();
    Q4Split sp{};
    const uint64_t G = a.n_head / a.n_head_kv;
    sp.chunks = (int)((G + kHeads - 1) / kHeads);
    const uint64_t units = a.n_q * a.n_head_kv * sp.chunks;
    int L = 0;
    while ((1ull << L) < a.page) ++L;
    sp.page_mul = (uint32_t)(((1ull << (31 + L)) + a.page - 1) / a.page);
    sp.page_shift = 31 + L;
    // enough CTAs to fill the GPU once, none with less than one stage per warp,
    // and none with more than 2048 tokens (a long sequence among short ones
    // would otherwise keep one CTA busy after the others are done)
    const uint64_t stages = (a.max_ctx + kCta - 1) / kCta;
    uint64_t want = std::max<uint64_t>(slots / units, (a.max_ctx + 2047) / 2048);
    want = std::max<uint64_t>(1, std::min<uint64_t>({want, stages, kMaxSplits}));
    sp.heads = (int)std::min<uint64_t>(kHeads, G);
    if (units * want > 0x7fffffffull) return cudaErrorInvalidConfiguration;
    if (want > 1 && want <= 8) {  // a cluster
        int c = 2;
        while (c < (int)want) c *= 2;
        sp.splits = c;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(units * c));
        cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)c;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, a, sp);
    }
    sp.splits = (int)want;
    if (want > 1) keep_pool_memory();
    if (want > 1)
        if (cudaError_t e = cudaMallocAsync(reinterpret_cast<void**>(&sp.scratch), units * want * sp.heads * (HD + 2) * 4, s))
            return e;
    kernel<<<(unsigned)(units * want), kWarps * 32, smem, s>>>(a, sp);
    cudaError_t e = cudaGetLastError();
    if (want > 1) {
        if (e == cudaSuccess) {
            e = launch_pdl(attn_q4_join_kernel<T, HD>, dim3((unsigned)units, (unsigned)sp.heads), dim3(256), 0, s, a, sp);
        }
        cudaFreeAsync(sp.scratch, s);
    }
    return e;
}
template <class T>
cudaError_t attn_decode(const AttnQ4Args& a, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) {
        if (a.n_head / a.n_head_kv <= 4) {
            if (a.hd == 64) return launch_decode<T, 64, true>(a, s);
            if (a.hd == 128) return launch_decode<T, 128, true>(a, s);
            return launch_decode<T, 256, true>(a, s);
        }
    }
    if (a.hd == 64) return launch_decode<T, 64, false>(a, s);
    if (a.hd == 128) return launch_decode<T, 128, false>(a, s);
    return launch_decode<T, 256, false>(a, s);
}

}  // namespace

cudaError_t attn_q4(int type, const AttnQ4Args& a, cudaStream_t s) {
    if (!a.n_q || !a.n_head) return cudaSuccess;
    const bool one = !a.q_start;
    if (type == kTypeF32) return one ? attn_decode<float>(a, s) : attn_rows<float>(a, s);
    if (type == kTypeF16) return one ? attn_decode<__half>(a, s) : attn_rows<__half>(a, s);
    return one ? attn_decode<__nv_bfloat16>(a, s) : attn_rows<__nv_bfloat16>(a, s);
}

}  // namespace mvb
