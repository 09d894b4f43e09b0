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

// two floats in a register pair: sm_100 multiplies and adds both with one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// A lane holds two 16-byte pieces of a head whose values turn with each other (or 16 neighbours where pairs lie side by side, or where nothing turns), head_dim / 16 lanes a head, so a
// norm is a few shuffles and a rotation needs no exchange.  Sine and cosine are the same for all heads of a token: a block takes `batch` tokens, computes their turns into shared memory
// (in 64 bits up to the fraction of a turn) while its first loads are under way, then walks the tokens' heads; values are copied behind them.  The bytes of the rows, queries and keys in and
// out, are the floor; what is near it is the issue rate, hence the paired arithmetic, weights as floats in shared memory and no division in the walk.
// Measured (graph of calls): 8 tokens 3.6 us (one round of memory, the turns, one round); 2,051 tokens of 24 / 4 gated heads of 256 with the store 15.5 (67 MB, floor 10.3); 8,192 of 40 / 8 heads of
// 128 37.5 = 5.4 TB/s (floor 30.9).  Blocks that stay and compute the next batch's turns ahead were slower (8,192 tokens 50 to 60 us before the arithmetic was paired).
constexpr int HEAD_THREADS = 256, HEAD_BATCH = 4;
template <bool INTERLEAVED>
__global__ void __launch_bounds__(HEAD_THREADS) head_norm_kernel(const __grid_constant__ gq_head_norm_args p, int batch, int group, int *status) {
    __shared__ float4 turns[HEAD_BATCH * 128];                 // [token][4][lane of a head]: of pairs 8 l + 2 e and the next, cos, cos, sin, sin
    __shared__ float4 weights[2][4][32];                       // queries, keys: [quarter of a lane's values][lane]
    __shared__ int64_t k_at[HEAD_BATCH], v_at[HEAD_BATCH];     // where a token's keys and values go, -1: nowhere
    const int D = p.head_dim, lanes = D / 16, half = p.rotary_dim / 2, turn_lanes = (half + 7) / 8, wide = p.gated ? 2 * D : D;
    const int l = threadIdx.x & (group - 1), sub = (int)threadIdx.x / group, per_turn = HEAD_THREADS / group;       // lane of the head, head of this turn
    const bool store = p.slots != nullptr, live = l < lanes, norms = p.q_norm || p.k_norm;
    const int heads = p.n_heads + p.n_kv_heads;
    const int64_t t0 = (int64_t)blockIdx.x * batch;
    const int tokens = (int)min((int64_t)batch, p.T - t0), items = tokens * heads;
    // the two pieces of this lane
    const bool turned = l < turn_lanes;
    const int c0 = INTERLEAVED ? 2 * l : turned ? l : half / 4 + 2 * (l - turn_lanes), c1 = INTERLEAVED || !turned ? c0 + 1 : l + turn_lanes;
    pdl_wait();
    pdl_trigger();

    const __nv_bfloat16 *rows = (const __nv_bfloat16 *)p.qkv + t0 * p.ld_qkv;
    const int64_t keys = (int64_t)p.n_heads * wide;
    auto load = [&](int t, int h, uint4 &x, uint4 &y) {
        const uint4 *src = (const uint4 *)(rows + t * p.ld_qkv + (h < p.n_heads ? h * wide : keys + (h - p.n_heads) * D));
        x = src[c0];
        y = src[c1];
    };
    int t = 0, h = sub;                                        // token and head of this turn
    while (h >= heads) { h -= heads; ++t; }
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (live && t < tokens) load(t, h, x, y);
    for (int i = threadIdx.x; i < tokens * half; i += HEAD_THREADS) {
        const int t = (unsigned)i / (unsigned)half, pair = i - t * half;
        const int64_t pos = p.positions_bytes == 8 ? ((const int64_t *)p.positions)[t0 + t] : ((const int32_t *)p.positions)[t0 + t];
        const float2 cs = turn_of(pos, p.inv_freq[pair], p.amplitude);
        float *at = (float *)(turns + (t * 4 + pair % 8 / 2) * turn_lanes + pair / 8) + pair % 2;
        at[0] = cs.x;
        at[2] = cs.y;
    }
    if (norms && sub < 2 && live) {
        const uint4 *w = (const uint4 *)(sub ? p.k_norm : p.q_norm);
        const uint4 one = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
        const uint4 w0 = w ? w[c0] : one, w1 = w ? w[c1] : one;
        const uint32_t v[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            weights[sub][i][l] = make_float4(__uint_as_float(v[2 * i] << 16), __uint_as_float(v[2 * i] & 0xffff0000u), __uint_as_float(v[2 * i + 1] << 16), __uint_as_float(v[2 * i + 1] & 0xffff0000u));
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

    for (int first = 0; first < items; first += per_turn) {    // whole warps stay for the shuffles
        const bool mine = live && t < tokens;
        const uint32_t raw[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        const int t_now = t, h_now = h;
        h += per_turn;
        while (h >= heads) { h -= heads; ++t; }
        if (live && t < tokens) load(t, h, x, y);
        uint64_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = pack2(__uint_as_float(raw[i] << 16), __uint_as_float(raw[i] & 0xffff0000u));
        const bool is_q = h_now < p.n_heads;
        if (norms) {
            uint64_t sq = mul2(u[0], u[0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) sq = fma2(u[i], u[i], sq);
            float sum = live ? unpack2(sq).x + unpack2(sq).y : 0.0f;
            for (int o = group / 2; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
            const bool has = is_q ? p.q_norm != nullptr : p.k_norm != nullptr;
            const float r = has ? rsqrtf(sum / D + p.eps) : 1.0f;
            const uint64_t rr = pack2(r, r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 w = weights[is_q ? 0 : 1][i][l];
                u[2 * i] = mul2(u[2 * i], mul2(rr, pack2(w.x, w.y)));
                u[2 * i + 1] = mul2(u[2 * i + 1], mul2(rr, pack2(w.z, w.w)));
            }
        }
        if (mine && turned) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 cs = turns[(t_now * 4 + e) * turn_lanes + l];
                if (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (l * 8 + 2 * e + j < half) {
                            const float c = j ? cs.y : cs.x, s = j ? cs.w : cs.z;
                            const float2 v = unpack2(u[2 * e + j]);
                            u[2 * e + j] = fma2(pack2(-v.y, v.x), pack2(s, s), mul2(u[2 * e + j], pack2(c, c)));
                        }
                } else {
                    const uint64_t c = pack2(cs.x, cs.y), s = pack2(cs.z, cs.w), a = u[e], b = u[e + 4];
                    u[e] = fma2(b, pack2(-cs.z, -cs.w), mul2(a, c));
                    u[e + 4] = fma2(a, s, mul2(b, c));
                }
            }
        }
        if (mine) {
            __nv_bfloat16 *dst;
            bool there = true;
            if (is_q) dst = (__nv_bfloat16 *)p.q_out + ((t0 + t_now) * p.n_heads + h_now) * D;
            else if (!store) dst = (__nv_bfloat16 *)p.k_out + ((t0 + t_now) * p.n_kv_heads + (h_now - p.n_heads)) * D;
            else {
                dst = (__nv_bfloat16 *)p.k_pages + k_at[t_now] + (h_now - p.n_heads) * p.k_strides[2];
                there = k_at[t_now] >= 0;
            }
            if (there) {
                uint32_t out[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 v = unpack2(u[i]);
                    const __nv_bfloat162 w = __floats2bfloat162_rn(v.x, v.y);
                    memcpy(&out[i], &w, 4);
                }
                ((uint4 *)dst)[c0] = make_uint4(out[0], out[1], out[2], out[3]);
                ((uint4 *)dst)[c1] = make_uint4(out[4], out[5], out[6], out[7]);
            }
        }
    }
    if (store) {
        const int pieces = p.n_kv_heads * D / 8;
        for (int t = 0; t < tokens; ++t) {
            if (v_at[t] < 0) continue;
            const uint4 *src = (const uint4 *)(rows + t * p.ld_qkv + keys + p.n_kv_heads * D);
            for (int i = threadIdx.x; i < pieces; i += HEAD_THREADS) {
                const int h = (unsigned)i / (unsigned)(D / 8), c = i - h * (D / 8);
                ((uint4 *)((__nv_bfloat16 *)p.v_pages + v_at[t] + h * p.v_strides[2]))[c] = src[i];
            }
        }
    }
}

// Heads that do not fall into pairs of 16-byte pieces (head_dim or a half-turned part that is no multiple of 16): one block to a token's head, a value at a time, the turn of its pair computed for each in 64 bits,
// which is what the time is.  2,000 tokens of 40 / 8 heads of 96 with 24 dimensions turned 64 us (floor 6.1; with 32 turned, in the kernel above, 13.7), 8 tokens 3.0.
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
    if (!is_q && p.slots) {
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
