// attn_q4.cu -- attention over the 4-bit paged cache (kv_q4.cuh).
//
//   out[r][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[r][h].k_t - m)
// over the first ctx_len[r] cached tokens of the row's sequence, in one pass
// with the running maximum m and sum.  A row with no tokens gives zeros; what
// lies past ctx_len, or on a page that does not exist, is never used.
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.cuh"
#include "kv_q4.cuh"

namespace mvb {

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

}  // namespace

cudaError_t attn_q4(int type, const AttnQ4Args& a, cudaStream_t s) {
    if (!a.n_q || !a.n_head) return cudaSuccess;
    if (type == kTypeF32) return attn_rows<float>(a, s);
    if (type == kTypeF16) return attn_rows<__half>(a, s);
    return attn_rows<__nv_bfloat16>(a, s);
}

}  // namespace mvb
