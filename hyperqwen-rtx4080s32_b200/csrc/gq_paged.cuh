// Attention of a sequence's newest tokens over its keys and values in the pages of a cache.
#pragma once
#include "gq_common.cuh"

namespace gq {

// one block of 128 threads to a token's query head: blocks of 128 keys, one running maximum and sum
__global__ void paged_attention_kernel(const gq_attention_args p, int *status) {
    __shared__ float q[256], w[128], red[4];
    __shared__ int bad;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, D = p.head_dim, kvh = h / (p.n_heads / p.n_kv_heads), lane = threadIdx.x & 31;
    int64_t seq = -1, first = 0, n = 0;
    if (p.q_starts) {
        for (int64_t s = 0; s < p.n_seqs; ++s)
            if (p.q_starts[s] <= t && t < p.q_starts[s + 1]) { seq = s; first = p.q_starts[s]; n = p.q_starts[s + 1] - first; break; }
    } else {
        n = p.T / p.n_seqs; seq = t / n; first = seq * n;
    }
    if (seq < 0) return;
    const int64_t seen = p.lens[seq] - n + (t - first) + 1;
    for (int i = threadIdx.x; i < D; i += 128) q[i] = __bfloat162float(((const __nv_bfloat16 *)p.q)[t * p.q_strides[0] + h * p.q_strides[1] + i]) * p.scale;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    float top = -INFINITY, total = 0.0f, o[2] = {0.0f, 0.0f};
    for (int64_t j0 = 0; j0 < seen; j0 += 128) {
        const int64_t j = j0 + threadIdx.x;
        float s = -INFINITY;
        if (j < seen) {
            const int64_t at = j / p.page_size, page = at < p.table_width ? p.page_table[seq * p.ld_table + at] : -1;
            if (page < 0 || page >= p.n_pages) bad = 1;
            else {
                const __nv_bfloat16 *k = (const __nv_bfloat16 *)p.k_pages + page * p.k_strides[0] + (j % p.page_size) * p.k_strides[1] + kvh * p.k_strides[2];
                s = 0.0f;
                for (int i = 0; i < D; ++i) s += q[i] * __bfloat162float(k[i]);
            }
        }
        float m = s;
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
        if (lane == 0) red[threadIdx.x / 32] = m;
        __syncthreads();
        if (bad) break;
        const float next = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), top), ref = next == -INFINITY ? 0.0f : next;
        const float keep = __expf(top - ref);
        w[threadIdx.x] = j < seen ? __expf(s - ref) : 0.0f;
        __syncthreads();
        top = next;
        total *= keep;
        o[0] *= keep; o[1] *= keep;
        for (int x = 0; x < 128 && j0 + x < seen; ++x) {
            total += w[x];
            const int64_t page = p.page_table[seq * p.ld_table + (j0 + x) / p.page_size];
            const __nv_bfloat16 *v = (const __nv_bfloat16 *)p.v_pages + page * p.v_strides[0] + ((j0 + x) % p.page_size) * p.v_strides[1] + kvh * p.v_strides[2];
            for (int i = 0; i < 2; ++i)
                if (threadIdx.x + 128 * i < D) o[i] += w[x] * __bfloat162float(v[threadIdx.x + 128 * i]);
        }
        __syncthreads();
    }
    if (bad && threadIdx.x == 0) atomicMax(status, GQ_DEV_BAD_SHAPE);
    for (int i = 0; i < 2; ++i) {
        const int d = threadIdx.x + 128 * i;
        if (d >= D) break;
        float v = bad ? __int_as_float(0x7fc00000) : total == 0.0f ? 0.0f : o[i] / total;
        if (p.gate) v /= 1.0f + __expf(-__bfloat162float(((const __nv_bfloat16 *)p.gate)[t * p.gate_strides[0] + h * p.gate_strides[1] + d]));
        ((__nv_bfloat16 *)p.out)[t * p.out_strides[0] + h * p.out_strides[1] + d] = __float2bfloat16_rn(v);
    }
}

}  // namespace gq
