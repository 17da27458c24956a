// rope_kv.cu -- rotary positions (half and interleaved pairs, part of the
// head, tables scaled for long contexts) and the append of rotated keys and of
// values to the paged cache in one launch.
//
// Rotation of pair (x0, x1) with the table's c, s of the row's position:
//   y0 = fma(x0, c, -(x1 s)),  y1 = fma(x0, s, x1 c)
// the roundings of the framework's other RoPE kernels, so the half layout over
// the whole head gives mv_rope's bits.  All of it is one pass over the data:
// memory bound for prompts, launch latency for decode steps.
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

// ---------------------------------------------------------------- apply
// Item j of a head: 2 V elements.  The first rot / 2V items rotate -- half
// layout: elements jV.. and rot/2 + jV..; interleaved: elements 2jV.. -- and
// both use table entries jV .. jV + V - 1.  The other items copy elements
// 2jV .. 2jV + 2V - 1.  Each item reads all it needs before it writes, so out
// may be x.
template <class T, int V, bool VEC>
__device__ __forceinline__ void rope_item(const T* __restrict__ x, T* out, int j, int rot, bool half_layout,
                                          const float* __restrict__ co, const float* __restrict__ si, bool live) {
    const int nr = rot / (2 * V);
    const int a = j < nr && half_layout ? j * V : 2 * j * V;
    const int b = j < nr && half_layout ? rot / 2 + j * V : 2 * j * V + V;
    float x0[V], x1[V];
    load_n<V, VEC>(x + a, x0);
    load_n<V, VEC>(x + b, x1);
    if (!live) {  // no such position: zeros
#pragma unroll
        for (int i = 0; i < V; ++i) x0[i] = x1[i] = 0.0f;
    } else if (j < nr) {
        float c[V], s[V];
        load_n<V, VEC>(co + j * V, c);
        load_n<V, VEC>(si + j * V, s);
        if (half_layout) {
#pragma unroll
            for (int i = 0; i < V; ++i) rotate(x0[i], x1[i], c[i], s[i]);
        } else if constexpr (V == 1) {
            rotate(x0[0], x1[0], c[0], s[0]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                rotate(x0[2 * i], x0[2 * i + 1], c[i], s[i]);
                rotate(x1[2 * i], x1[2 * i + 1], c[V / 2 + i], s[V / 2 + i]);
            }
        }
    }
    store_n<V, VEC>(out + a, x0);
    store_n<V, VEC>(out + b, x1);
}

// The q part of one row (and the whole of mv_rope_apply): items of all heads
// spread over the CTAs `part` of `parts`.
template <class T, int V, bool VEC>
__device__ __forceinline__ void rope_row(const RopeApplyArgs& a, int64_t r, int part, int parts) {
    const int per = (int)a.hd / (2 * V), items = (int)a.n_head * per;
    const int p = a.pos[r];
    const bool live = p >= 0 && (!a.rot || (uint64_t)p < a.n_pos);
    const int half = (int)a.rot / 2;
    const float* co = a.cos_t + (live ? (int64_t)p * half : 0);
    const float* si = a.sin_t + (live ? (int64_t)p * half : 0);
    const T* x = static_cast<const T*>(a.x) + r * (int64_t)a.x_stride;
    T* out = static_cast<T*>(a.out) + r * (int64_t)a.out_stride;
    for (int i = part * (int)blockDim.x + (int)threadIdx.x; i < items; i += parts * (int)blockDim.x) {
        const int h = i / per, j = i % per;
        rope_item<T, V, VEC>(x + h * (int64_t)a.x_head_stride, out + h * (int64_t)a.out_head_stride, j, (int)a.rot,
                             a.layout == 0, co, si, live);
    }
}

template <class T, int V, bool VEC>
__global__ void __launch_bounds__(256) rope_apply_kernel(RopeApplyArgs a) {
    rope_row<T, V, VEC>(a, blockIdx.x, blockIdx.y, gridDim.y);
}

// --------------------------------------------------------------- append
// 8 dimensions d .. d + 7 of a k head, rotated; the partners are read from the
// row itself (the same lines: L1), so no exchange between threads is needed.
template <class T, bool VEC>
__device__ __forceinline__ void rotated8(const T* __restrict__ x, int d, int rot, bool half_layout,
                                         const float* __restrict__ co, const float* __restrict__ si, float (&y)[8]) {
    load_n<8, VEC>(x + d, y);
    if (d >= rot) return;
    const int half = rot / 2;
    if constexpr (VEC) {  // rot % 16 == 0: the 8 are all rotated, all in one half
        if (half_layout) {
            const bool second = d >= half;
            const int i = second ? d - half : d;
            float o[8], c[8], s[8];
            load_n<8, true>(x + (second ? i : d + half), o);
            load_n<8, true>(co + i, c);
            load_n<8, true>(si + i, s);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                y[k] = second ? __fmaf_rn(o[k], s[k], __fmul_rn(y[k], c[k]))
                              : __fmaf_rn(y[k], c[k], -__fmul_rn(o[k], s[k]));
        } else {
            float c[4], s[4];
            load_n<4, true>(co + d / 2, c);
            load_n<4, true>(si + d / 2, s);
#pragma unroll
            for (int k = 0; k < 4; ++k) rotate(y[2 * k], y[2 * k + 1], c[k], s[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int e = d + k;
            if (e >= rot) continue;
            const bool second = half_layout ? e >= half : (e & 1);
            const int i = half_layout ? (second ? e - half : e) : e / 2;
            const float o = to_f32(x[half_layout ? (second ? i : e + half) : (e ^ 1)]);
            y[k] = second ? __fmaf_rn(o, si[i], __fmul_rn(y[k], co[i])) : __fmaf_rn(y[k], co[i], -__fmul_rn(o, si[i]));
        }
    }
}

// The cache slot of row r, or -1 where the row is skipped: a negative
// position, one outside the table of angles or the block table, a sequence or
// page that does not exist.
__device__ __forceinline__ int64_t kv_slot_page(const KvRows& k, int64_t r, int* slot) {
    const int p = k.pos[r];
    const int s = k.row_is_seq ? (int)r : k.seq ? k.seq[r] : 0;
    if (p < 0 || (uint64_t)p >= k.max_pages * k.page || s < 0 || (uint64_t)s >= k.n_seq) return -1;
    const int64_t pg = k.block_table[(int64_t)s * (int64_t)k.max_pages + p / (int)k.page];
    *slot = p % (int)k.page;
    return pg >= 0 && pg < (int64_t)k.n_pages ? pg : -1;
}

template <class T, bool VEC, int KVT>
__global__ void __launch_bounds__(256) rope_kv_append_kernel(RopeAppendArgs a) {
    const int64_t r = blockIdx.x;
    if (a.ctx_out && blockIdx.y == 0 && threadIdx.x == 0) a.ctx_out[r] = a.rows.pos[r] + 1;
    if ((int)blockIdx.y < a.q_parts) {
        rope_row<T, VEC ? 16 / (int)sizeof(T) : 1, VEC>(a.q, r, blockIdx.y, a.q_parts);
        return;
    }
    // 8 dimensions per thread: K heads, then V heads (a multiple of 32 items
    // each when the type has 32-element blocks, so a block's 4 lanes stay together)
    const int hd = (int)a.hd, per = hd / 8, items = 2 * (int)a.n_head_kv * per;
    int slot = 0;
    const int64_t pg = kv_slot_page(a.rows, r, &slot);
    const int p = a.rows.pos[r];
    if (pg < 0 || (a.rot && (uint64_t)p >= a.n_pos)) return;
    const int half = (int)a.rot / 2;
    const float* co = a.cos_t + (int64_t)p * half;
    const float* si = a.sin_t + (int64_t)p * half;
    const int parts = (int)gridDim.y - a.q_parts, part = (int)blockIdx.y - a.q_parts;
    if constexpr (KVT == 2) {
        // one scale per token over all kv_dim elements: a CTA takes the K or V
        // row, its largest magnitude first, then the row again (from L1/L2)
        __shared__ float red[8];
        const bool is_v = part;
        const T* x = static_cast<const T*>(is_v ? a.v : a.k) + r * (int64_t)(is_v ? a.v_stride : a.k_stride);
        const int n = (int)a.n_head_kv * per;
        float m = 0.0f, y[8];
        auto take = [&](int i) {
            const T* h = x + (i / per) * (int64_t)(is_v ? a.v_head_stride : a.k_head_stride);
            const int d = i % per * 8;
            if (is_v) load_n<8, VEC>(h + d, y);
            else rotated8<T, VEC>(h, d, (int)a.rot, a.layout == 0, co, si, y);
        };
        for (int i = threadIdx.x; i < n; i += 256) {
            take(i);
#pragma unroll
            for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(y[k]));
        }
        m = warp_max(m);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        m = red[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = fmaxf(m, red[w]);
        const float sc = m > 0.0f ? m / 127.0f : 1.0f;
        const int64_t row = pg * (int64_t)a.rows.page + slot;
        int8_t* dst = static_cast<int8_t*>(is_v ? a.v_pages : a.k_pages) + row * (int64_t)(a.n_head_kv * a.hd);
        for (int i = threadIdx.x; i < n; i += 256) {
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
    } else {
        // every lane of a warp takes the same number of turns (the quantisers'
        // shuffles need all 32): lanes past the end do the first block, store nothing
        for (int base = part * 256; base < items; base += parts * 256) {
            const bool in = base + (int)threadIdx.x < items;
            if (KVT <= 1 && !in) break;
            const int i = in ? base + (int)threadIdx.x : (int)threadIdx.x & 3;
            const bool is_v = i >= items / 2;
            const int k = is_v ? i - items / 2 : i, head = k / per, d = k % per * 8;
            float y[8];
            if (is_v) {
                load_n<8, VEC>(static_cast<const T*>(a.v) + r * (int64_t)a.v_stride + head * (int64_t)a.v_head_stride + d, y);
            } else {
                rotated8<T, VEC>(static_cast<const T*>(a.k) + r * (int64_t)a.k_stride + head * (int64_t)a.k_head_stride, d,
                                 (int)a.rot, a.layout == 0, co, si, y);
            }
            void* pages = is_v ? a.v_pages : a.k_pages;
            if constexpr (KVT == kKvQ4) {
                uint16_t sc;
                const uint32_t w = q4_quantise8(y, &sc);
                const int nb = hd / 32, b = d / 32, t = d / 8 % 4;
                const int64_t tok = (pg * (int64_t)a.n_head_kv + head) * (int64_t)a.rows.page + slot;
                if (in) {
                    static_cast<uint32_t*>(pages)[tok * (hd / 8) + t * nb + b] = w;
                    if (t == 0) static_cast<uint16_t*>(is_v ? a.v_scales : a.k_scales)[tok * nb + b] = sc;
                }
            } else {
                const int64_t at = ((pg * (int64_t)a.rows.page + slot) * (int64_t)a.n_head_kv + head) * hd + d;
                if constexpr (KVT == 3) {
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
                        *reinterpret_cast<uint2*>(static_cast<int8_t*>(pages) + at) = o.w;
                        if (d % 32 == 0) static_cast<float*>(is_v ? a.v_scales : a.k_scales)[at / 32] = dd;
                    }
                } else if (in) {
                    if constexpr (KVT == 0) store_n<8, true>(static_cast<float*>(pages) + at, y);
                    else store_n<8, true>(static_cast<__half*>(pages) + at, y);
                }
            }
        }
    }
}

// ----------------------------------------------------------------- read
// Rows of one pool as out[row][kv head][hd]; a skipped row reads zeros.
template <class T>
__global__ void __launch_bounds__(256) kv_read_kernel(KvReadArgs a) {
    const int64_t r = blockIdx.x;
    const int hd = (int)a.hd, per = hd / 8, items = (int)a.n_head_kv * per;
    int slot = 0;
    const int64_t pg = kv_slot_page(a.rows, r, &slot);
    T* out = static_cast<T*>(a.out) + r * (int64_t)items * 8;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < items; i += gridDim.y * 256) {
        const int head = i / per, d = i % per * 8;
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = 0.0f;
        if (pg >= 0) {
            const int64_t row = pg * (int64_t)a.rows.page + slot, at = row * (int64_t)items * 8 + (int64_t)i * 8;
            if (a.kv_type == 0) {
                load_n<8, true>(static_cast<const float*>(a.pages) + at, y);
            } else if (a.kv_type == 1) {
                load_n<8, true>(static_cast<const __half*>(a.pages) + at, y);
            } else if (a.kv_type == kKvQ4) {
                const int nb = hd / 32, b = d / 32, t = d / 8 % 4;
                const int64_t tok = (pg * (int64_t)a.n_head_kv + head) * (int64_t)a.rows.page + slot;
                const uint32_t w = static_cast<const uint32_t*>(a.pages)[tok * (hd / 8) + t * nb + b];
                const float s = bf16_bits_to_f32(static_cast<const uint16_t*>(a.scales)[tok * nb + b]);
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = (float)((int)((w >> (4 * k)) & 15u) - 8) * s;
            } else {
                const float* sc = static_cast<const float*>(a.scales);
                const float s = a.kv_type == 2 ? sc[row] : sc[at / 32];
                const int8_t* q = static_cast<const int8_t*>(a.pages) + at;
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = (float)q[k] * s;
            }
        }
        store_n<8, true>(out + (int64_t)i * 8, y);
    }
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

template <class T, bool VEC, int KVT>
cudaError_t launch_append(const RopeAppendArgs& a, unsigned parts, cudaStream_t s) {
    rope_kv_append_kernel<T, VEC, KVT><<<dim3((unsigned)a.n_rows, (unsigned)a.q_parts + parts), 256, 0, s>>>(a);
    return cudaGetLastError();
}
template <class T, bool VEC>
cudaError_t append_kv(const RopeAppendArgs& a, unsigned parts, cudaStream_t s) {
    switch (a.kv_type) {
        case 0: return launch_append<T, VEC, 0>(a, parts, s);
        case 1: return launch_append<T, VEC, 1>(a, parts, s);
        case 2: return launch_append<T, VEC, 2>(a, parts, s);
        case 3: return launch_append<T, VEC, 3>(a, parts, s);
        default: return launch_append<T, VEC, kKvQ4>(a, parts, s);
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
    const uint64_t v = vec ? 16 / type_size(type) : 1, items = a.n_head * (a.hd / (2 * v));
    const dim3 grid((unsigned)rows, (unsigned)std::min<uint64_t>((items + 255) / 256, 65535));
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, s>>>(a);
        return cudaGetLastError();
    };
    if (type == kTypeF32) return vec ? go(rope_apply_kernel<float, 4, true>) : go(rope_apply_kernel<float, 1, false>);
    if (type == kTypeF16) return vec ? go(rope_apply_kernel<__half, 8, true>) : go(rope_apply_kernel<__half, 1, false>);
    return vec ? go(rope_apply_kernel<__nv_bfloat16, 8, true>) : go(rope_apply_kernel<__nv_bfloat16, 1, false>);
}

cudaError_t rope_kv_append(int type, const RopeAppendArgs& args, cudaStream_t s) {
    RopeAppendArgs a = args;
    if (!a.n_rows) return cudaSuccess;
    const uint64_t e = type_size(type), v = 16 / e;
    const bool kv_vec = a.rot % 16 == 0 && a.k_stride % v == 0 && a.v_stride % v == 0 && a.k_head_stride % v == 0 &&
                        a.v_head_stride % v == 0 && aligned16(a.k) && aligned16(a.v) && aligned16(a.cos_t) &&
                        aligned16(a.sin_t);
    const bool vec = kv_vec && (!a.q.n_head || rope_vec_ok(a.q, type));
    const uint64_t qi = a.q.n_head * (a.hd / (vec ? 2 * v : 2)), ki = 2 * a.n_head_kv * (a.hd / 8);
    a.q_parts = (int)((qi + 255) / 256);
    const unsigned parts = a.kv_type == 2 ? 2u : (unsigned)((ki + 255) / 256);
    if (type == kTypeF32) return vec ? append_kv<float, true>(a, parts, s) : append_kv<float, false>(a, parts, s);
    if (type == kTypeF16) return vec ? append_kv<__half, true>(a, parts, s) : append_kv<__half, false>(a, parts, s);
    return vec ? append_kv<__nv_bfloat16, true>(a, parts, s) : append_kv<__nv_bfloat16, false>(a, parts, s);
}

cudaError_t kv_read(int type, const KvReadArgs& a, uint64_t rows, cudaStream_t s) {
    if (!rows) return cudaSuccess;
    const dim3 grid((unsigned)rows, (unsigned)((a.n_head_kv * (a.hd / 8) + 255) / 256));
    if (type == kTypeF32) kv_read_kernel<float><<<grid, 256, 0, s>>>(a);
    else if (type == kTypeF16) kv_read_kernel<__half><<<grid, 256, 0, s>>>(a);
    else kv_read_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace mvb
