// Queries and keys as qkv_proj wrote them -> normalised by head, rotated by position, keys and values into the pages of a cache.
#pragma once
#include "gq_common.cuh"

namespace gq {

// cos and sin of position * inv_freq radians, times the amplitude.  The angle is reduced to a fraction of a turn in 64 bits (a float's 24 bits
// are spent on the whole turns of a far position), then 24 bits of that fraction are plenty.
__device__ __forceinline__ float2 turn_of(int64_t position, double inv_freq, float amplitude) {
    const double turns = (double)position * (inv_freq * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * amplitude, s * amplitude);
}

// one block to a token's head: queries, keys, then values if there are pages
__global__ void head_norm_kernel(const gq_head_norm_args p, int *status) {
    __shared__ float u[512];
    __shared__ float part[32];
    const int D = p.head_dim, wide = p.gated ? 2 * D : D, head = blockIdx.y;
    const int64_t t = blockIdx.x;
    const bool is_q = head < p.n_heads, is_k = !is_q && head < p.n_heads + p.n_kv_heads;
    const int h = is_q ? head : is_k ? head - p.n_heads : head - p.n_heads - p.n_kv_heads;
    const __nv_bfloat16 *src = (const __nv_bfloat16 *)p.qkv + t * p.ld_qkv +
                               (is_q ? (int64_t)h * wide : (int64_t)p.n_heads * wide + (int64_t)(is_k ? h : h + p.n_kv_heads) * D);
    __nv_bfloat16 *dst = is_q ? (__nv_bfloat16 *)p.q_out + (t * p.n_heads + h) * D : (__nv_bfloat16 *)p.k_out + (t * p.n_kv_heads + h) * D;
    if (!is_q && p.k_pages) {
        const int64_t slot = p.slots_bytes == 8 ? ((const int64_t *)p.slots)[t] : ((const int32_t *)p.slots)[t];
        if (slot < 0) return;
        const int64_t page = slot / p.page_size, row = slot % p.page_size;
        if (page >= p.n_pages) {
            if (threadIdx.x == 0) atomicMax(status, GQ_DEV_BAD_SHAPE);
            return;
        }
        const int64_t *st = is_k ? p.k_strides : p.v_strides;
        dst = (__nv_bfloat16 *)(is_k ? p.k_pages : p.v_pages) + page * st[0] + row * st[1] + h * st[2];
    }
    if (!is_q && !is_k) {
        for (int i = threadIdx.x; i < D; i += blockDim.x) dst[i] = src[i];
        return;
    }
    const __nv_bfloat16 *w = (const __nv_bfloat16 *)(is_q ? p.q_norm : p.k_norm);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) { u[i] = __bfloat162float(src[i]); sum += u[i] * u[i]; }
    if (w) {
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int i = 0; i < blockDim.x / 32; ++i) sum += part[i];
        const float r = rsqrtf(sum / D + p.eps);
        for (int i = threadIdx.x; i < D; i += blockDim.x) u[i] *= r * __bfloat162float(w[i]);
    }
    __syncthreads();
    const int64_t pos = p.positions_bytes == 8 ? ((const int64_t *)p.positions)[t] : ((const int32_t *)p.positions)[t];
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        float v = u[i];
        if (i < p.rotary_dim) {
            const int half = p.rotary_dim / 2, pair = p.interleaved ? i / 2 : i % half;
            const bool second = p.interleaved ? (i & 1) : i >= half;
            const int other = p.interleaved ? i ^ 1 : second ? i - half : i + half;
            const float2 cs = turn_of(pos, p.inv_freq[pair], p.amplitude);
            v = second ? v * cs.x + u[other] * cs.y : v * cs.x - u[other] * cs.y;
        }
        dst[i] = __float2bfloat16_rn(v);
    }
}

}  // namespace gq
