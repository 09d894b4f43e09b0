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

// A lane holds two 16-byte pieces of a head whose values turn with each other (or 16 neighbours where pairs lie side by side, or where nothing turns), head_dim / 16 lanes a head, so a
// norm is a few shuffles and a rotation needs no exchange.  Sine and cosine are the same for all heads of a token: a block takes `batch` tokens, computes their turns into shared memory
// (in 64 bits up to the fraction of a turn) while its first loads are under way, then walks the tokens' heads.  Bound by the bytes of the rows: queries and keys in and out.
constexpr int HEAD_THREADS = 256, HEAD_BATCH = 4;
template <bool INTERLEAVED>
__global__ void __launch_bounds__(HEAD_THREADS) head_norm_kernel(const __grid_constant__ gq_head_norm_args p, int batch, int group, int *status) {
    __shared__ float4 turns[HEAD_BATCH * 128];                 // [token][4][lane of a head]: cos, sin of pairs 8 l + 2 e and the next
    __shared__ int64_t k_at[HEAD_BATCH], v_at[HEAD_BATCH];     // where a token's keys and values go, -1: nowhere
    const int D = p.head_dim, lanes = D / 16, half = p.rotary_dim / 2, turn_lanes = (half + 7) / 8, wide = p.gated ? 2 * D : D;
    const int l = threadIdx.x % group, sub = threadIdx.x / group, per_turn = HEAD_THREADS / group;       // lane of the head, head of this turn
    const bool store = p.k_pages != nullptr, live = l < lanes;
    const int heads = p.n_heads + (store ? 2 : 1) * p.n_kv_heads;
    const int64_t t0 = (int64_t)blockIdx.x * batch;
    const int tokens = (int)min((int64_t)batch, p.T - t0), items = tokens * heads;
    // the two pieces of this lane
    const bool turned = l < turn_lanes;
    const int c0 = INTERLEAVED ? 2 * l : turned ? l : half / 4 + 2 * (l - turn_lanes), c1 = INTERLEAVED || !turned ? c0 + 1 : l + turn_lanes;
    pdl_wait();
    pdl_trigger();

    auto load = [&](int item, uint4 (&x)[2]) {
        const int t = item / heads, h = item - t * heads;
        const int64_t at = (t0 + t) * p.ld_qkv + (h < p.n_heads ? (int64_t)h * wide : (int64_t)p.n_heads * wide + (int64_t)(h - p.n_heads) * D);
        const uint4 *src = (const uint4 *)((const __nv_bfloat16 *)p.qkv + at);
        x[0] = src[c0];
        x[1] = src[c1];
    };
    uint4 x[2];
    int item = sub;
    if (live && item < items) load(item, x);
    uint4 wq[2], wk[2];
    if (live) {
        if (p.q_norm) { wq[0] = ((const uint4 *)p.q_norm)[c0]; wq[1] = ((const uint4 *)p.q_norm)[c1]; }
        if (p.k_norm) { wk[0] = ((const uint4 *)p.k_norm)[c0]; wk[1] = ((const uint4 *)p.k_norm)[c1]; }
    }
    for (int i = threadIdx.x; i < tokens * half; i += HEAD_THREADS) {
        const int t = i / half, pair = i - t * half;
        const int64_t pos = p.positions_bytes == 8 ? ((const int64_t *)p.positions)[t0 + t] : ((const int32_t *)p.positions)[t0 + t];
        ((float2 *)turns)[(t * 4 + pair % 8 / 2) * turn_lanes * 2 + pair / 8 * 2 + pair % 2] = turn_of(pos, p.inv_freq[pair], p.amplitude);
    }
    if (store && threadIdx.x >= HEAD_THREADS - HEAD_BATCH && (int)threadIdx.x - (HEAD_THREADS - HEAD_BATCH) < tokens) {
        const int t = threadIdx.x - (HEAD_THREADS - HEAD_BATCH);
        const int64_t slot = p.slots_bytes == 8 ? ((const int64_t *)p.slots)[t0 + t] : ((const int32_t *)p.slots)[t0 + t], page = slot < 0 ? -1 : slot / p.page_size;
        const bool ok = page >= 0 && page < p.n_pages;
        const int64_t row = slot - page * p.page_size;
        k_at[t] = ok ? page * p.k_strides[0] + row * p.k_strides[1] : -1;
        v_at[t] = ok ? page * p.v_strides[0] + row * p.v_strides[1] : -1;
        if (page >= p.n_pages) atomicMax(status, GQ_DEV_BAD_SHAPE);
    }
    __syncthreads();

    for (; item - sub < items; item += per_turn) {             // whole warps stay for the shuffles
        const bool mine = live && item < items;
        uint4 next[2];
        if (live && item + per_turn < items) load(item + per_turn, next);
        const int t = item / heads, h = item - t * heads;
        const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv_heads, plain = !is_q && !is_k;
        float u[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w = i < 4 ? (&x[0].x)[i] : (&x[1].x)[i - 4];
            u[2 * i] = mine ? __uint_as_float(w << 16) : 0.0f;
            u[2 * i + 1] = mine ? __uint_as_float(w & 0xffff0000u) : 0.0f;
        }
        if (p.q_norm || p.k_norm) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += u[i] * u[i];
            for (int o = group / 2; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
            if (mine && (is_q ? p.q_norm != nullptr : is_k && p.k_norm)) {
                const float r = rsqrtf(sum / D + p.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = is_q ? (i < 4 ? (&wq[0].x)[i] : (&wq[1].x)[i - 4]) : (i < 4 ? (&wk[0].x)[i] : (&wk[1].x)[i - 4]);
                    u[2 * i] *= r * __uint_as_float(w << 16);
                    u[2 * i + 1] *= r * __uint_as_float(w & 0xffff0000u);
                }
            }
        }
        if (mine && turned && !plain) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 cs = turns[(t * 4 + e) * turn_lanes + l];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int pair = 2 * e + j;                // of this lane's eight
                    if (INTERLEAVED && l * 8 + pair >= half) continue;
                    const float c = j ? cs.z : cs.x, s = j ? cs.w : cs.y;
                    float &a = u[INTERLEAVED ? 2 * pair : pair], &b = u[INTERLEAVED ? 2 * pair + 1 : pair + 8];
                    const float was = a;
                    a = was * c - b * s;
                    b = b * c + was * s;
                }
            }
        }
        if (mine) {
            const int kv = plain ? h - p.n_heads - p.n_kv_heads : h - p.n_heads;
            __nv_bfloat16 *dst;
            if (is_q) dst = (__nv_bfloat16 *)p.q_out + ((t0 + t) * p.n_heads + h) * D;
            else if (!store) dst = (__nv_bfloat16 *)p.k_out + ((t0 + t) * p.n_kv_heads + kv) * D;
            else if (is_k) dst = (__nv_bfloat16 *)p.k_pages + k_at[t] + kv * p.k_strides[2];
            else dst = (__nv_bfloat16 *)p.v_pages + v_at[t] + kv * p.v_strides[2];
            if (is_q || !store || k_at[t] >= 0) {
                uint4 y[2];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(u[2 * i], u[2 * i + 1]);
                    memcpy(i < 4 ? &(&y[0].x)[i] : &(&y[1].x)[i - 4], &v, 4);
                }
                if (plain) { y[0] = x[0]; y[1] = x[1]; }        // values as they are, NaNs among them
                ((uint4 *)dst)[c0] = y[0];
                ((uint4 *)dst)[c1] = y[1];
            }
        }
        x[0] = next[0];
        x[1] = next[1];
    }
}

// Heads that do not fall into pairs of 16-byte pieces (head_dim or a half-turned part that is no multiple of 16): one block to a token's head, a value at a time
__global__ void head_norm_any_kernel(const gq_head_norm_args p, int *status) {
    __shared__ float u[512];
    __shared__ float part[32];
    const int D = p.head_dim, wide = p.gated ? 2 * D : D, head = blockIdx.y;
    const int64_t t = blockIdx.x;
    pdl_wait();
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
