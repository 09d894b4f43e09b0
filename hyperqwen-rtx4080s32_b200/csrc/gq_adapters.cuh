// Low-rank adapters beside a shared projection: out = base + scale * B (A x) for each row's own adapter.
#pragma once
#include "gq_common.cuh"

namespace gq {

struct LowRankParams {
    const __nv_bfloat16 *base, *x, *a, *b;
    const float *scales;
    const void *ids;
    __nv_bfloat16 *out;
    float *inner;                // [M, n_shards * rank]
    int64_t K, ld_base, ldx, ld_out, n_total;
    int64_t edges[9];            // first column of each shard, and the end
    int M, n_shards, n_adapters, rank, wide_ids;
};

__device__ __forceinline__ int64_t id_at(const void *ids, int wide, int64_t i) { return wide ? ((const int64_t *)ids)[i] : ((const int32_t *)ids)[i]; }

// A x: one warp to an inner value, which it scales
__global__ void low_rank_inner_kernel(const LowRankParams p) {
    const int cols = p.n_shards * p.rank, lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (at >= (int64_t)p.M * cols) return;
    const int64_t m = at / cols;
    const int c = (int)(at % cols);
    const int64_t id = id_at(p.ids, p.wide_ids, m);
    if (id < 0 || id >= p.n_adapters) return;
    const __nv_bfloat16 *x = p.x + m * p.ldx, *a = p.a + (id * cols + c) * p.K;
    float sum = 0.0f;
    for (int64_t k = lane; k < p.K; k += 32) sum += __bfloat162float(x[k]) * __bfloat162float(a[k]);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) p.inner[at] = sum * p.scales[id * p.n_shards + c / p.rank];
}

// base + B (A x): one thread to a column
__global__ void low_rank_outer_kernel(const LowRankParams p, int *status) {
    const int64_t m = blockIdx.x, n = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    const int64_t id = id_at(p.ids, p.wide_ids, m);
    if (n >= p.n_total) return;
    float v = __bfloat162float(p.base[m * p.ld_base + n]);
    if (id >= 0 && id < p.n_adapters) {
        int s = 0;
        while (n >= p.edges[s + 1]) ++s;
        const float *t = p.inner + (m * p.n_shards + s) * p.rank;
        const __nv_bfloat16 *b = p.b + (id * p.n_total + n) * p.rank;
        for (int r = 0; r < p.rank; ++r) v += __bfloat162float(b[r]) * t[r];
    } else if (id != -1) {
        v = __int_as_float(0x7fc00000);
        if (n == 0) atomicMax(status, GQ_DEV_BAD_SHAPE);
    }
    p.out[m * p.ld_out + n] = __float2bfloat16_rn(v);
}

}  // namespace gq
