// kv_q4.cuh -- the 4-bit KV block (MV_KV_Q4_0) and element conversions shared
// by the append, read and attention kernels.
//
// A block is 32 consecutive dimensions of one head of one token:
//   mx = the element of largest magnitude (the first of equals, with its sign)
//   d  = bf16(mx / -8), round to nearest even
//   n  = clamp(floor(x * (1/d) + 8.5), 0, 15)        value = (n - 8) * d
// d has 8 significant bits and n - 8 at most 4, so a value has at most 11: it
// is exact in fp16 up to a power of two, and the tensor cores take the cache's
// values without another rounding.  A block with a NaN or an infinity gets
// d = NaN, so every value of it is NaN; one whose largest magnitude is below
// 2^-100 is stored as zeros (1/d would leave the fp32 range).
//
// Layout of a pool, K and V alike:
//   nibbles [page][kv head][token of the page][hd / 2 bytes]
//   scales  [page][kv head][token of the page][hd / 32] bf16
// so one head's tokens of a page are one contiguous run.  A token's 32-bit
// words are ordered [4][hd / 32]: word (t, b) holds dimensions 32 b + 8 t .. +7,
// lowest nibble first.  A 16-byte piece at hd 128 is then word t of every
// block, which is what one lane of an m16n8k16 fragment multiplies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "common.cuh"
#include "tc.cuh"

namespace mvb {

// activation types of the entry points (GGML type ids)
constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 30;
constexpr int kKvQ4 = 4;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements <-> fp32 registers; VEC: the address is aligned for
// 16-byte accesses (32-bit types: two of them for N = 8).
template <int N, bool VEC, class T>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
    if constexpr (VEC && sizeof(T) == 4 && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    } else if constexpr (VEC && sizeof(T) == 2 && N == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
            x[2 * i] = to_f32(reinterpret_cast<const T&>(lo));
            x[2 * i + 1] = to_f32(reinterpret_cast<const T&>(hi));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f32(p[i]);
    }
}
template <int N, bool VEC, class T>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
    if constexpr (VEC && sizeof(T) == 4 && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else if constexpr (VEC && sizeof(T) == 2 && N == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T a = from_f32<T>(x[2 * i]), b = from_f32<T>(x[2 * i + 1]);
            w[i] = (uint32_t)reinterpret_cast<const uint16_t&>(a) |
                   ((uint32_t)reinterpret_cast<const uint16_t&>(b) << 16);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// Quantises a block held by 4 consecutive lanes, 8 dimensions each (lane t of
// the four: dimensions 8 t .. + 7).  Returns this lane's word; *scale gets the
// bf16 bits.  Every lane of the warp calls it.
__device__ __forceinline__ uint32_t q4_quantise8(const float (&x)[8], uint16_t* scale) {
    // the largest magnitude; its first holder's sign.  A NaN anywhere makes
    // `bad` non-zero (x - x is 0 only for finite x).
    float mx = x[0], bad = x[0] - x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        if (fabsf(x[i]) > fabsf(mx)) mx = x[i];
        bad += x[i] - x[i];
    }
    bad = bad == 0.0f ? 0.0f : 1.0f;
    const int t = (int)(threadIdx.x & 3u);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, mx, o);
        bad += __shfl_xor_sync(0xffffffffu, bad, o);
        const float a = fabsf(mx), b = fabsf(other);
        // equal magnitudes: the lower lane's (lower dimensions) sign
        if (b > a || (b == a && (t & o))) mx = other;
    }
    const bool zero = fabsf(mx) < 7.8886090522101181e-31f;  // 2^-100
    const __nv_bfloat16 db = __float2bfloat16_rn(zero ? 0.0f : __fdiv_rn(mx, -8.0f));
    const float d = __bfloat162float(db);
    const float inv = zero ? 0.0f : __frcp_rn(d);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = floorf(__fadd_rn(__fmul_rn(x[i], inv), 8.5f));
        w |= (uint32_t)(int)fminf(fmaxf(r, 0.0f), 15.0f) << (4 * i);
    }
    *scale = bad != 0.0f ? (uint16_t)0x7fc0u : reinterpret_cast<const uint16_t&>(db);
    return bad != 0.0f ? 0x88888888u : w;
}

// ------------------------------------------------- arithmetic on the blocks
// Half-precision queries: factor on the weights for what their cut to 11 bits
// (tf32, by the tensor core) takes off on average, 1 + 2^-11 / (2 ln 2), their
// mantissas being log-uniform.
constexpr float kCut = 1.00035225f;
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
// Nibbles 0 and 4 of x as the fp16 numbers n - 8, or nibbles 1 and 5 as 16 (n -
// 8): ORed into 1024 they are 1024 + n, or 1024 + 16 n, and one subtraction is
// exact.  (As fp16 subnormals n 2^-24, without it, the tensor core aligned its
// sum to their exponent field, 2^-14, and scores lost 4 bits.)
__device__ __forceinline__ uint32_t nib_lo(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    const __half2 h = __hadd2(reinterpret_cast<const __half2&>(r), __float2half2_rn(-1032.0f));
    return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint32_t nib_hi(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(x));
    const __half2 h = __hadd2(reinterpret_cast<const __half2&>(r), __float2half2_rn(-1152.0f));
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
// Nibbles I, I + 1 of x as (n - 8) 16^I, (n - 8) 16^(I + 1) in fp32: each is
// masked in place and ORed into the mantissa of 2^23, and one packed addition
// takes `bias`, the pair 2^23 + 8 16^I, .., off.  The pair are neighbours in
// the MMA's A registers (rows g, g + 8).
template <int I>
__device__ __forceinline__ void values2(uint32_t x, uint64_t bias, float& v0, float& v1) {
    uint32_t u0, u1;
    asm("lop3.b32 %0, %1, %2, 0x4b000000, 0xea;" : "=r"(u0) : "r"(x), "n"(0xf << (4 * I)));
    asm("lop3.b32 %0, %1, %2, 0x4b000000, 0xea;" : "=r"(u1) : "r"(x), "n"(0xf0 << (4 * I)));
    unpair(f2_add(pair(__uint_as_float(u0), __uint_as_float(u1)), bias), v0, v1);
}
// A pair of constants that stays in registers (the compiler would build it anew at every use).
__device__ __forceinline__ uint64_t held_pair(float lo, float hi) {
    uint64_t r;
    asm volatile("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t bits16) { return __uint_as_float(bits16 << 16); }

}  // namespace mvb
