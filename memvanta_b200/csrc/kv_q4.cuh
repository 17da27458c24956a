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
#include <type_traits>

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

// N consecutive elements, held as loaded (half types in half the registers)
// until they are used.  VEC: the address is aligned for 16-byte accesses.
template <class T, int N, bool VEC>
struct Held {
    static constexpr int kBytes = N * (int)sizeof(T), kWords = kBytes / 4;
    static constexpr bool kWide = VEC && kBytes % 16 == 0;
    uint32_t w[kWide ? kWords : 1];
    T v[kWide ? 1 : N];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
                w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) =
                    make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = v[i];
        }
    }
    __device__ __forceinline__ void get(float (&x)[N]) const {
        if constexpr (kWide && sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = __uint_as_float(w[i]);
        } else if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
                x[2 * i] = to_f32(reinterpret_cast<const T&>(lo));
                x[2 * i + 1] = to_f32(reinterpret_cast<const T&>(hi));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = to_f32(v[i]);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[N]) {
        if constexpr (kWide && sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = __float_as_uint(x[i]);
        } else if constexpr (kWide && std::is_same<T, __half>::value) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(h);
            }
        } else if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(h);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = from_f32<T>(x[i]);
        }
    }
    __device__ __forceinline__ void zero() {
        const float none[N] = {};
        set(none);
    }
};
template <int N, bool VEC, class T>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
    Held<T, N, VEC> h;
    h.load(p);
    h.get(x);
}
template <int N, bool VEC, class T>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
    Held<T, N, VEC> h;
    h.set(x);
    h.store(p);
}

// Two floats in a register pair, and their sums (tc.cuh: products).  The compiler
// may join a packed product and the packed sum that it feeds into one rounding.
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

// Quantises a block held by 4 consecutive lanes, 8 dimensions each (lane t of
// the four: dimensions 8 t .. + 7).  Returns this lane's word; *scale gets the
// bf16 bits.  Every lane of the warp calls it.
__device__ __forceinline__ uint32_t q4_quantise8(const float (&x)[8], uint16_t* scale) {
    // the element of largest magnitude: the greater of the largest and the
    // smallest, and of equal ones the first
    float hi = x[0], lo = x[0];
    uint64_t bad2 = 0;  // 0, or NaN of a NaN or an infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) hi = fmaxf(hi, x[i]), lo = fminf(lo, x[i]);
#pragma unroll
    for (int i = 0; i < 8; i += 2) bad2 = tc::f2_fma(pair(x[i], x[i + 1]), 0, bad2);
    float bad, bad_hi;
    unpair(bad2, bad, bad_hi);
    bad += bad_hi;
    float mx = hi > -lo ? hi : lo;
    if (hi == -lo) {
#pragma unroll
        for (int i = 7; i >= 0; --i)
            if (fabsf(x[i]) == hi) mx = x[i];
    }
    const float inf = __uint_as_float(0x7f800000u);
    if (bad != 0.0f) mx = inf;
    const int t = (int)(threadIdx.x & 3u);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, mx, o);
        const float a = fabsf(mx), b = fabsf(other);
        // equal magnitudes: the lower lane's (lower dimensions) sign
        if (b > a || (b == a && (t & o))) mx = other;
    }
    if (fabsf(mx) == inf) {
        *scale = 0x7fc0u;
        return 0x88888888u;
    }
    const bool zero = fabsf(mx) < 7.8886090522101181e-31f;  // 2^-100
    const __nv_bfloat16 db = __float2bfloat16_rn(zero ? 0.0f : __fmul_rn(mx, -0.125f));
    const float inv = zero ? 0.0f : __frcp_rn(__bfloat162float(db));
    // |x (1/d)| is at most 8 (1 + 2^-8), so the sum lies in (0, 17): only 15 needs
    // a clamp.  floor by adding 2^23 rounded down: the low bits are n, and the
    // eight exponents that the shifts leave in the word add up to 0xfb000000
    // (the products one by one: a packed product and a packed sum came out as one
    // rounding, which moves values that lie on a boundary)
    const uint64_t mid = pair(8.5f, 8.5f);
    uint32_t w = 0u - 0xfb000000u;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float r0, r1;
        unpair(f2_add(pair(__fmul_rn(x[i], inv), __fmul_rn(x[i + 1], inv)), mid), r0, r1);
        w += __float_as_uint(__fadd_rd(fminf(r0, 15.5f), 8388608.0f)) << (4 * i);
        w += __float_as_uint(__fadd_rd(fminf(r1, 15.5f), 8388608.0f)) << (4 * i + 4);
    }
    *scale = reinterpret_cast<const uint16_t&>(db);
    return w;
}

// ------------------------------------------------- arithmetic on the blocks
// Half-precision queries: a weight such that its first 11 bits, which are what the
// tensor core takes of a tf32 operand, are the nearest 11 (ties away from zero).
__device__ __forceinline__ float near11(float x) { return __uint_as_float(__float_as_uint(x) + 0x1000u); }
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
