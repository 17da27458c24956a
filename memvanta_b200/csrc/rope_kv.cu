// rope_kv.cu -- rotary positions (half and interleaved pairs, part of the
// head, tables scaled for long contexts) and the append of rotated keys and of
// values to the paged cache in one launch.
//
// Rotation of pair (x0, x1) with the table's c, s of the row's position:
//   y0 = fma(x0, c, -(x1 s)),  y1 = fma(x0, s, x1 c)
// the roundings of the framework's other RoPE kernels, so the half layout over
// the whole head gives mv_rope's bits.
//
// All of it is one pass over the data.  Measured (back-to-back launches; a plain
// copy of 67 MB takes 22.9 us):
//   rotation, 4,093 rows of 32 heads x 128 fp32, 134 MB         22.7 us  5.9 TB/s
//   rotation, 8,191 rows of 32 heads x 128 bf16, 134 MB         27.7 us  4.8 TB/s
//   append to F16, 2,048 rows, 32 + 2 x 8 heads x 128 fp16       9.3 us  5.4 TB/s
//   append to Q4_0, 4,093 rows, 32 + 2 x 32 heads x 128 fp32    67.9 us  4.2 TB/s
//   rotation or append of 64 rows                          2.0 and 3.3 us
//   reading 4,093 rows x 32 x 128 of Q4_0 back as fp16         10.9 us  4.0 TB/s
// The Q4_0 append is bound by instructions: 500 for 16 dimensions of K and V, half
// of them the block's scale and the rounding of its nibbles (63% of the issue
// slots are taken, 36% of the memory's time).  So is the read-back: 16 instructions
// a value, 75% of the issue slots, 64% of the integer pipe.  Small calls are a
// launch and three loads that wait on one another (position, page, angle).
// Tried: a thread for several heads, so that the row's part is done once
// (113 to 127 us with its reads, 101 without: fewer threads hide less), lines
// asked for into L2 a wave ahead (no change), 8-byte accesses for half types
// (29 us for the 27.7).
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.cuh"
#include "kv_q4.cuh"

namespace mvb {

namespace {

__device__ __forceinline__ void rotate(float& x0, float& x1, float c, float s) {
    const float y0 = __fmaf_rn(x0, c, -__fmul_rn(x1, s));
    x1 = __fmaf_rn(x0, s, __fmul_rn(x1, c));
    x0 = y0;
}

// --------------------------------------------------------------- tables
// cos/sin of pos * inv_freq in double (a float angle of position 131071 is off
// by up to 2^-8), rounded once.  Runs once per table.
__global__ void rope_table_kernel(RopeScaling r, int half, int64_t n_pos, const float* __restrict__ factors,
                                  float* __restrict__ cos_t, float* __restrict__ sin_t) {
    const double kTwoPi = 6.283185307179586476925;
    for (int64_t k = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; k < n_pos * half;
         k += (int64_t)gridDim.x * blockDim.x) {
        const int i = (int)(k % half);
        const int64_t p = k / half;
        double inv = pow(r.theta, -(double)i / (double)half);
        if (factors) inv /= (double)factors[i];
        double mul = 1.0;
        if (r.kind == 1) {
            inv /= r.factor;
        } else if (r.kind == 2) {
            // interpolate the dimensions that turn less than beta_slow times over
            // the original context, keep those that turn more than beta_fast
            // times, a linear ramp over the dimension index between
            const double two_half = 2.0 * half, lt = 2.0 * log(r.theta);
            const double d_fast = two_half * log(r.orig_ctx / (r.beta_fast * kTwoPi)) / lt;
            const double d_slow = two_half * log(r.orig_ctx / (r.beta_slow * kTwoPi)) / lt;
            const double lo = fmax(floor(d_fast), 0.0), hi = fmin(ceil(d_slow), two_half - 1.0);
            const double ramp = fmin(fmax(((double)i - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
            inv = inv / r.factor * ramp + inv * (1.0 - ramp);
            mul = r.attn_factor > 0.0 ? r.attn_factor : (r.factor > 1.0 ? 0.1 * log(r.factor) + 1.0 : 1.0);
        } else if (r.kind == 3) {
            // by wavelength: short ones kept, long ones divided, a smooth step between
            const double turns = r.orig_ctx * inv / kTwoPi;  // turns over the original context
            const double keep = fmin(fmax((turns - r.beta_slow) / (r.beta_fast - r.beta_slow), 0.0), 1.0);
            inv = (1.0 - keep) * inv / r.factor + keep * inv;
        }
        const double a = (double)p * inv;
        cos_t[k] = (float)(cos(a) * mul);
        sin_t[k] = (float)(sin(a) * mul);
    }
}

// ---------------------------------------------------------------- items
// A row is `items` pieces of work, a few dimensions of a head each, `per` to a
// head, and a thread does one: what hides the memory's latency is many threads
// with their loads issued at once.  A block holds several rows, or a row takes
// several blocks.
constexpr int kThreads = 256;

struct Div {  // n / d for n < 2^31: umulhi(2 n, mul) >> shift
    uint32_t d, mul;
    int shift;
};
Div div_by(uint64_t d) {
    int L = 0;
    while ((1ull << L) < d) ++L;
    return {(uint32_t)d, (uint32_t)(((1ull << (31 + L)) + d - 1) / d), L};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const Div& v) { return __umulhi(n << 1, v.mul) >> v.shift; }

struct Items {
    Div per, items, parts;  // parts: blocks of a row
    int rows;               // rows of a block
    uint64_t blocks;
};
Items items_of(uint64_t n_rows, uint64_t heads, uint64_t per) {
    Items t;
    const uint64_t items = heads * per, parts = (items + kThreads - 1) / kThreads;
    t.per = div_by(per), t.items = div_by(items), t.parts = div_by(parts);
    t.rows = (int)std::max<uint64_t>(1, kThreads / items);
    t.blocks = parts > 1 ? n_rows * parts : (n_rows + t.rows - 1) / t.rows;
    return t;
}
// This thread's row, head and piece of the head; false: none.
__device__ __forceinline__ bool place(const Items& t, uint32_t block, int64_t n_rows, int64_t* row, int* head,
                                      int* piece) {
    uint32_t i = threadIdx.x;
    bool has;
    if (t.parts.d > 1) {
        const uint32_t r = block / t.parts;
        i += (block - r * t.parts.d) * kThreads;
        *row = r;
        has = i < t.items.d;
    } else {
        const uint32_t in = i / t.items;
        *row = (int64_t)block * t.rows + in;
        i -= in * t.items.d;
        has = (int)in < t.rows && *row < n_rows;
    }
    *head = (int)(i / t.per);
    *piece = (int)i - *head * (int)t.per.d;
    return has;
}

// ---------------------------------------------------------------- apply
// Piece j of a head: 2 V elements.  The first rot / 2V pieces rotate -- half
// layout: elements jV.. and rot/2 + jV..; interleaved: elements 2jV.. -- and
// both use table entries jV .. jV + V - 1.  The others copy elements 2jV .. 2jV +
// 2V - 1.  Each piece is read before it is written, so out may be x.
template <class T, int V, bool VEC>
__device__ __forceinline__ void rope_piece(const RopeApplyArgs& a, const Items& t, uint32_t block, int64_t n_rows) {
    int64_t r;
    int h, j;
    if (!place(t, block, n_rows, &r, &h, &j)) return;
    const int rot = (int)a.rot, half = rot / 2;
    const bool turns = j < rot / (2 * V), half_layout = a.layout == 0;
    const int p = a.pos[r];
    const int e = turns && half_layout ? j * V : 2 * j * V, gap = turns && half_layout ? half : V;
    const T* x = static_cast<const T*>(a.x) + r * (int64_t)a.x_stride + h * (int64_t)a.x_head_stride + e;
    Held<T, V, VEC> x0, x1;
    x0.load(x);
    x1.load(x + gap);
    if (p < 0 || (rot && (uint64_t)p >= a.n_pos)) {  // no such position: zeros
        x0.zero();
        x1.zero();
    } else if (turns) {
        float c[V], s[V], y0[V], y1[V];
        load_n<V, VEC>(a.cos_t + (int64_t)p * half + j * V, c);
        load_n<V, VEC>(a.sin_t + (int64_t)p * half + j * V, s);
        x0.get(y0);
        x1.get(y1);
        if (half_layout || V == 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) rotate(y0[k], y1[k], c[k], s[k]);
        } else if constexpr (V > 1) {
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                rotate(y0[2 * k], y0[2 * k + 1], c[k], s[k]);
                rotate(y1[2 * k], y1[2 * k + 1], c[V / 2 + k], s[V / 2 + k]);
            }
        }
        x0.set(y0);
        x1.set(y1);
    }
    T* out = static_cast<T*>(a.out) + r * (int64_t)a.out_stride + h * (int64_t)a.out_head_stride + e;
    x0.store(out);
    x1.store(out + gap);
}

template <class T, int V, bool VEC>
__global__ void __launch_bounds__(kThreads, 5) rope_apply_kernel(RopeApplyArgs a, Items t, int64_t n_rows) {
    rope_piece<T, V, VEC>(a, t, blockIdx.x, n_rows);
}

// --------------------------------------------------------------- append
// 8 dimensions d .. d + 7 of a k head.  take8: what the row holds of them and of
// their partners (the same lines: L1).  angles8: the row's table entries.  Then
// rotate8.  VEC (rot % 16 == 0, so the 8 rotate together) in the half layout: y and o
// are elements of the first and the second half, and with the factors swapped for
// the second half's results, (c, -s) or (s, c), both come from fma(y, c, o s).
template <class T, bool VEC>
__device__ __forceinline__ void take8(const T* __restrict__ x, int d, int rot, bool half_layout, Held<T, 8, VEC>& y,
                                      Held<T, 8, VEC>& o) {
    const int half = rot / 2;
    if (VEC && half_layout && d < rot) {
        y.load(d >= half ? x - half : x);
        o.load(d >= half ? x : x + half);
        return;
    }
    y.load(x);
    if constexpr (!VEC) {
        if (d >= rot || !half_layout) return;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (d + k < rot) o.v[k] = d + k >= half ? x[k - half] : x[k + half];
    }
}
// Entry k of c, s is dimension d + k's (half layout) or pair k's (interleaved, 4 of them).
template <bool VEC>
__device__ __forceinline__ void angles8(const float* __restrict__ co, const float* __restrict__ si, int d, int rot,
                                        bool half_layout, float (&c)[8], float (&s)[8]) {
    if (d >= rot) return;
    const int half = rot / 2;
    if (half_layout) {
        if constexpr (VEC) {
            const bool second = d >= half;
            load_n<8, true>(second ? si + (d - half) : co + d, c);
            load_n<8, true>(second ? co + (d - half) : si + d, s);
            if (!second) {
#pragma unroll
                for (int k = 0; k < 8; ++k) s[k] = -s[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (d + k >= rot) continue;
                const int i = d + k >= half ? d + k - half : d + k;
                c[k] = co[i], s[k] = si[i];
            }
        }
    } else if constexpr (VEC) {
        const float4 c4 = *reinterpret_cast<const float4*>(co + d / 2);
        const float4 s4 = *reinterpret_cast<const float4*>(si + d / 2);
        c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
        s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (d + 2 * k < rot) c[k] = co[d / 2 + k], s[k] = si[d / 2 + k];
    }
}
template <class T, bool VEC>
__device__ __forceinline__ void rotate8(float (&y)[8], const Held<T, 8, VEC>& partner, const float (&c)[8],
                                        const float (&s)[8], int d, int rot, bool half_layout) {
    if (d >= rot) return;
    if (half_layout) {
        float o[8];
        partner.get(o);
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                unpair(tc::f2_fma(pair(y[k], y[k + 1]), pair(c[k], c[k + 1]),
                              tc::f2_mul(pair(o[k], o[k + 1]), pair(s[k], s[k + 1]))),
                       y[k], y[k + 1]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (d + k < rot)
                    y[k] = d + k >= rot / 2 ? __fmaf_rn(o[k], s[k], __fmul_rn(y[k], c[k]))
                                            : __fmaf_rn(y[k], c[k], -__fmul_rn(o[k], s[k]));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (VEC || d + 2 * k < rot) rotate(y[2 * k], y[2 * k + 1], c[k], s[k]);
    }
}

// The cache slot of row r, or -1 where the row is skipped: a negative
// position, one outside the table of angles or the block table, a sequence or
// page that does not exist.
__device__ __forceinline__ int64_t kv_slot_page(const KvRows& k, const Div& page, int64_t r, int* slot) {
    const int p = k.pos[r];
    const int s = k.row_is_seq ? (int)r : k.seq ? k.seq[r] : 0;
    if (p < 0 || (uint64_t)p >= k.max_pages * k.page || s < 0 || (uint64_t)s >= k.n_seq) return -1;
    const uint32_t pi = (uint32_t)p / page;
    const int64_t pg = k.block_table[(int64_t)s * (int64_t)k.max_pages + pi];
    *slot = p - (int)(pi * page.d);
    return pg >= 0 && pg < (int64_t)k.n_pages ? pg : -1;
}

// Where 8 dimensions of a head lie in a pool, and their block's scale: indices
// of words (Q4_0) or elements, and of scales.
struct Spot {
    int64_t at, scale;
};
template <int KVT>
__device__ __forceinline__ Spot spot_of(int64_t pg, int slot, int page, int heads, int head, int hd, int d) {
    Spot s;
    if constexpr (KVT == kKvQ4) {
        const int nb = hd / 32;
        const int64_t tok = (pg * heads + head) * page + slot;
        s.scale = tok * nb + d / 32;
        s.at = tok * (hd / 8) + d / 8 % 4 * nb + d / 32;
    } else {
        s.at = ((pg * page + slot) * heads + head) * hd + d;
        s.scale = s.at / 32;
    }
    return s;
}
// 8 dimensions as the cache holds them (lanes in fours hold a block's 32; all of
// the warp call it, `in`: this one stores).
template <int KVT>
__device__ __forceinline__ void put8(const float (&y)[8], void* pages, void* scales, const Spot& s, int d, bool in) {
    if constexpr (KVT == kKvQ4) {
        uint16_t sc;
        const uint32_t w = q4_quantise8(y, &sc);
        if (in) {
            static_cast<uint32_t*>(pages)[s.at] = w;
            if (d % 32 == 0) static_cast<uint16_t*>(scales)[s.scale] = sc;
        }
    } else if constexpr (KVT == 3) {
        float m = fabsf(y[0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, fabsf(y[e]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const float dd = m > 0.0f ? m / 127.0f : 1.0f, inv = 1.0f / dd;
        union {
            int8_t b[8];
            uint2 w;
        } o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.b[e] = (int8_t)(int)fminf(fmaxf(roundf(y[e] * inv), -127.0f), 127.0f);
        if (in) {
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(pages) + s.at) = o.w;
            if (d % 32 == 0) static_cast<float*>(scales)[s.scale] = dd;
        }
    } else if (in) {
        if constexpr (KVT == 0) store_n<8, true>(static_cast<float*>(pages) + s.at, y);
        else store_n<8, true>(static_cast<__half*>(pages) + s.at, y);
    }
}

// Queries and cache rows in turn, block by block, while both last: the first wait
// for memory, the others for instructions (72.9 us one after the other, 67.9 so).
__device__ __forceinline__ bool rotates(uint32_t block, uint32_t q, uint32_t kv, uint32_t* index) {
    const uint32_t both = 2 * min(q, kv);
    *index = block < both ? block / 2 : block - both / 2;
    return block < both ? block % 2 : q > kv;
}

// 8 dimensions of K and of V of a head to a thread.
template <class T, bool VEC, int KVT>
__global__ void __launch_bounds__(kThreads, 4) rope_kv_append_kernel(RopeAppendArgs a, Items tq, Items t, Div page) {
    uint32_t block;
    if (rotates(blockIdx.x, (uint32_t)tq.blocks, (uint32_t)t.blocks, &block)) {
        rope_piece<T, VEC ? 16 / (int)sizeof(T) : 1, VEC>(a.q, tq, block, (int64_t)a.n_rows);
        return;
    }
    const int hd = (int)a.hd, rot = (int)a.rot;
    const bool half_layout = a.layout == 0;
    int64_t r;
    int h, j;
    // (a block's scale is found by shuffles, so that a thread without work does
    // row 0's first block, and stores nothing)
    const bool has = place(t, block, (int64_t)a.n_rows, &r, &h, &j);
    if (!has) r = 0, h = 0, j &= 3;
    const int d = j * 8;
    const int p = a.rows.pos[r];
    Held<T, 8, VEC> hk, ho, hv;
    take8(static_cast<const T*>(a.k) + r * (int64_t)a.k_stride + h * (int64_t)a.k_head_stride + d, d, rot, half_layout,
          hk, ho);
    hv.load(static_cast<const T*>(a.v) + r * (int64_t)a.v_stride + h * (int64_t)a.v_head_stride + d);
    if (a.ctx_out && has && h == 0 && j == 0) a.ctx_out[r] = p + 1;
    float c[8], s[8], y[8];
    const bool angles = p >= 0 && (uint64_t)p < a.n_pos;
    if (angles) {
        const int64_t at = (int64_t)p * (rot / 2);
        angles8<VEC>(a.cos_t + at, a.sin_t + at, d, rot, half_layout, c, s);
    }
    int slot = 0;
    const int64_t pg = kv_slot_page(a.rows, page, r, &slot);
    const bool in = has && pg >= 0 && (!rot || angles);
    const Spot spot = spot_of<KVT>(pg, slot, (int)a.rows.page, (int)a.n_head_kv, h, hd, d);
    hk.get(y);
    rotate8(y, ho, c, s, d, rot, half_layout);
    put8<KVT>(y, a.k_pages, a.k_scales, spot, d, in);
    hv.get(y);
    put8<KVT>(y, a.v_pages, a.v_scales, spot, d, in);
}

// Q8: one scale per token over all kv_dim elements.  A block takes a row's K or
// V: its largest magnitude first, then the row again (from L1/L2).
template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_kv_append_q8_kernel(RopeAppendArgs a, Items tq, Div page) {
    uint32_t block;
    if (rotates(blockIdx.x, (uint32_t)tq.blocks, 2 * (uint32_t)a.n_rows, &block)) {
        rope_piece<T, VEC ? 16 / (int)sizeof(T) : 1, VEC>(a.q, tq, block, (int64_t)a.n_rows);
        return;
    }
    __shared__ float red[kThreads / 32];
    const int64_t r = block / 2;
    const bool is_v = block % 2;
    const int hd = (int)a.hd, per = hd / 8, n = (int)a.n_head_kv * per, rot = (int)a.rot;
    const int p = a.rows.pos[r];
    if (a.ctx_out && !is_v && threadIdx.x == 0) a.ctx_out[r] = p + 1;
    int slot = 0;
    const int64_t pg = kv_slot_page(a.rows, page, r, &slot);
    if (pg < 0 || (rot && (uint64_t)p >= a.n_pos)) return;
    const float* co = a.cos_t + (int64_t)p * (rot / 2);
    const float* si = a.sin_t + (int64_t)p * (rot / 2);
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + r * (int64_t)(is_v ? a.v_stride : a.k_stride);
    float y[8];
    auto take = [&](int i) {
        const T* h = x + (i / per) * (int64_t)(is_v ? a.v_head_stride : a.k_head_stride);
        const int d = i % per * 8;
        if (is_v) {
            load_n<8, VEC>(h + d, y);
        } else {
            Held<T, 8, VEC> own, o;
            float c[8], s[8];
            take8(h + d, d, rot, a.layout == 0, own, o);
            own.get(y);
            angles8<VEC>(co, si, d, rot, a.layout == 0, c, s);
            rotate8(y, o, c, s, d, rot, a.layout == 0);
        }
    };
    float m = 0.0f;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        take(i);
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(y[k]));
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
    const float sc = m > 0.0f ? m / 127.0f : 1.0f;
    const int64_t row = pg * (int64_t)a.rows.page + slot;
    int8_t* dst = static_cast<int8_t*>(is_v ? a.v_pages : a.k_pages) + row * (int64_t)(a.n_head_kv * a.hd);
    for (int i = threadIdx.x; i < n; i += kThreads) {
        take(i);
        union {
            int8_t b[8];
            uint2 w;
        } o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.b[k] = (int8_t)(int)fminf(fmaxf(roundf(y[k] / sc), -127.0f), 127.0f);
        *reinterpret_cast<uint2*>(dst + (int64_t)i * 8) = o.w;
    }
    if (threadIdx.x == 0) static_cast<float*>(is_v ? a.v_scales : a.k_scales)[row] = sc;
}

// ----------------------------------------------------------------- read
// Rows of one pool as out[row][kv head][hd]; a skipped row reads zeros.  A thread
// takes 8 dimensions, of Q4_0 B times that: the same quarter of B blocks that
// follow one another, whose words and scales do too (4,093 rows x 32 x 128 to fp16:
// 10.9 us with B = 2, 15.2 us with 1).
template <class T, int KVT, int B>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvReadArgs a, Items t, Div page, int64_t n_rows) {
    int64_t r;
    int h, j;
    if (!place(t, blockIdx.x, n_rows, &r, &h, &j)) return;
    const int hd = (int)a.hd, H = (int)a.n_head_kv, d = B == 1 ? j * 8 : j / 4 * (32 * B) + j % 4 * 8;
    int slot = 0;
    const int64_t pg = kv_slot_page(a.rows, page, r, &slot);
    float y[B][8];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int k = 0; k < 8; ++k) y[b][k] = 0.0f;
    if (pg >= 0) {
        const Spot s = spot_of<KVT>(pg, slot, (int)a.rows.page, H, h, hd, d);
        if constexpr (KVT == 0) {
            load_n<8, true>(static_cast<const float*>(a.pages) + s.at, y[0]);
        } else if constexpr (KVT == 1) {
            load_n<8, true>(static_cast<const __half*>(a.pages) + s.at, y[0]);
        } else if constexpr (KVT == kKvQ4) {
            uint32_t w[B];
            float sc[B];
            if constexpr (B == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint32_t*>(a.pages) + s.at);
                const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.scales) + s.scale);
                w[0] = v.x, w[1] = v.y;
                sc[0] = __uint_as_float(u << 16), sc[1] = __uint_as_float(u & 0xffff0000u);
            } else {
                w[0] = static_cast<const uint32_t*>(a.pages)[s.at];
                sc[0] = bf16_bits_to_f32(static_cast<const uint16_t*>(a.scales)[s.scale]);
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int k = 0; k < 8; ++k) y[b][k] = (float)((int)(w[b] >> (4 * k) & 15u) - 8) * sc[b];
        } else {
            const float sc = static_cast<const float*>(a.scales)[KVT == 2 ? pg * (int64_t)a.rows.page + slot : s.scale];
            const int8_t* q = static_cast<const int8_t*>(a.pages) + s.at;
#pragma unroll
            for (int k = 0; k < 8; ++k) y[0][k] = (float)q[k] * sc;
        }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) store_n<8, true>(static_cast<T*>(a.out) + (r * H + h) * hd + d + 32 * b, y[b]);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
uint64_t type_size(int type) { return type == kTypeF32 ? 4 : 2; }

// Whether every access of a rotation can be a 16-byte one.
bool rope_vec_ok(const RopeApplyArgs& a, int type) {
    const uint64_t v = 16 / type_size(type);
    return a.rot % 16 == 0 && a.hd % 16 == 0 && (a.hd - a.rot) % (2 * v) == 0 && a.rot % (2 * v) == 0 &&
           a.x_stride % v == 0 && a.out_stride % v == 0 && a.x_head_stride % v == 0 && a.out_head_stride % v == 0 &&
           aligned16(a.x) && aligned16(a.out) && aligned16(a.cos_t) && aligned16(a.sin_t);
}

constexpr uint64_t kMaxGrid = 0x7fffffff;

template <class T, bool VEC>
cudaError_t append_kv(const RopeAppendArgs& a, cudaStream_t s) {
    constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
    Items tq{};
    if (a.q.n_head) tq = items_of(a.n_rows, a.q.n_head, a.hd / (2 * V));
    const Items t = items_of(a.n_rows, a.n_head_kv, a.hd / 8);
    const Div page = div_by(a.rows.page);
    const uint64_t grid = tq.blocks + (a.kv_type == 2 ? 2 * a.n_rows : t.blocks);
    if (grid > kMaxGrid) return cudaErrorInvalidConfiguration;
    switch (a.kv_type) {
        case 0: rope_kv_append_kernel<T, VEC, 0><<<(unsigned)grid, kThreads, 0, s>>>(a, tq, t, page); break;
        case 1: rope_kv_append_kernel<T, VEC, 1><<<(unsigned)grid, kThreads, 0, s>>>(a, tq, t, page); break;
        case 2: rope_kv_append_q8_kernel<T, VEC><<<(unsigned)grid, kThreads, 0, s>>>(a, tq, page); break;
        case 3: rope_kv_append_kernel<T, VEC, 3><<<(unsigned)grid, kThreads, 0, s>>>(a, tq, t, page); break;
        default: rope_kv_append_kernel<T, VEC, kKvQ4><<<(unsigned)grid, kThreads, 0, s>>>(a, tq, t, page);
    }
    return cudaGetLastError();
}
template <class T>
cudaError_t read_kv(const KvReadArgs& a, uint64_t rows, cudaStream_t s) {
    const bool two = a.kv_type == kKvQ4 && a.hd % 64 == 0;
    const Items t = items_of(rows, a.n_head_kv, a.hd / (two ? 16 : 8));
    const Div page = div_by(a.rows.page);
    if (t.blocks > kMaxGrid) return cudaErrorInvalidConfiguration;
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)t.blocks, kThreads, 0, s>>>(a, t, page, (int64_t)rows);
        return cudaGetLastError();
    };
    switch (a.kv_type) {
        case 0: return go(kv_read_kernel<T, 0, 1>);
        case 1: return go(kv_read_kernel<T, 1, 1>);
        case 2: return go(kv_read_kernel<T, 2, 1>);
        case 3: return go(kv_read_kernel<T, 3, 1>);
        default: return two ? go(kv_read_kernel<T, kKvQ4, 2>) : go(kv_read_kernel<T, kKvQ4, 1>);
    }
}

}  // namespace

cudaError_t rope_table(const RopeScaling& r, uint64_t rot, uint64_t n_pos, const float* factors, float* cos_t,
                       float* sin_t, cudaStream_t s) {
    const uint64_t n = n_pos * (rot / 2);
    if (!n) return cudaSuccess;
    const uint64_t blocks = (n + 255) / 256;
    rope_table_kernel<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(r, (int)(rot / 2), (int64_t)n_pos,
                                                                                  factors, cos_t, sin_t);
    return cudaGetLastError();
}

cudaError_t rope_apply(int type, const RopeApplyArgs& a, uint64_t rows, cudaStream_t s) {
    if (!rows || !a.n_head || !a.hd) return cudaSuccess;
    const bool vec = rope_vec_ok(a, type);
    const Items t = items_of(rows, a.n_head, a.hd / (2 * (vec ? 16 / type_size(type) : 1)));
    if (t.blocks > kMaxGrid) return cudaErrorInvalidConfiguration;
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)t.blocks, kThreads, 0, s>>>(a, t, (int64_t)rows);
        return cudaGetLastError();
    };
    if (type == kTypeF32) return vec ? go(rope_apply_kernel<float, 4, true>) : go(rope_apply_kernel<float, 1, false>);
    if (type == kTypeF16) return vec ? go(rope_apply_kernel<__half, 8, true>) : go(rope_apply_kernel<__half, 1, false>);
    return vec ? go(rope_apply_kernel<__nv_bfloat16, 8, true>) : go(rope_apply_kernel<__nv_bfloat16, 1, false>);
}

cudaError_t rope_kv_append(int type, const RopeAppendArgs& a, cudaStream_t s) {
    if (!a.n_rows) return cudaSuccess;
    const uint64_t v = 16 / type_size(type);
    const bool kv_vec = a.rot % 16 == 0 && a.k_stride % v == 0 && a.v_stride % v == 0 && a.k_head_stride % v == 0 &&
                        a.v_head_stride % v == 0 && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos_t) &&
                        aligned16(a.sin_t);
    const bool vec = kv_vec && (!a.q.n_head || rope_vec_ok(a.q, type));
    if (type == kTypeF32) return vec ? append_kv<float, true>(a, s) : append_kv<float, false>(a, s);
    if (type == kTypeF16) return vec ? append_kv<__half, true>(a, s) : append_kv<__half, false>(a, s);
    return vec ? append_kv<__nv_bfloat16, true>(a, s) : append_kv<__nv_bfloat16, false>(a, s);
}

cudaError_t kv_read(int out_type, const KvReadArgs& a, uint64_t rows, cudaStream_t s) {
    if (!rows) return cudaSuccess;
    if (out_type == kTypeF32) return read_kv<float>(a, rows, s);
    if (out_type == kTypeF16) return read_kv<__half>(a, rows, s);
    return read_kv<__nv_bfloat16>(a, rows, s);
}

}  // namespace mvb
