// Low-rank adapters beside a shared projection: out = base + scale * B (A x) for each row's own adapter.
//
// Rows are taken in tiles of 64; a block sorts its tile's rows by adapter, and every adapter that occurs multiplies its own rows only, so no row's sums ever hold another adapter's numbers and
// rows of one adapter need not stand together.  Two launches: the inner products A x, their sums over parts of K left in the workspace, and the outer products B (A x) with the addition.
// Both read bf16 operands from global memory straight into the fragments of mma.sync m16n8k16: any order of k serves as long as both operands have the same, so a lane takes 8
// neighbours (16 bytes) where the instruction names scattered ones.  Bound by bytes: in decode those of the adapters (latency below a few MB), in prefill those of base and out;
// the ranks are too small for tcgen05's 128 rows to be filled.
#pragma once
#include "gq_bf16.cuh"

namespace gq {

constexpr int LR_ROWS = 64, LR_THREADS = 256, LR_WARPS = LR_THREADS / 32;

struct LowRankParams {
    const __nv_bfloat16 *base, *x, *a, *b;
    const float *scales;
    const void *ids;
    __nv_bfloat16 *out;
    float *inner;                // workspace: [parts][M][n_shards * ranks], scaled
    int *status;
    int64_t ld_base, ldx, ld_out, n_total;
    int64_t edges[9];            // first column of each shard, and the end
    int M, K, n_shards, n_adapters, rank, ranks, parts, wide_ids;       // ranks: the rank as the outer products see it, 16, 32, 64 or 128
    int cols, vec;               // columns of an outer block; base and out can be read and written 16 bytes at a time
};

__device__ __forceinline__ int64_t id_at(const void *ids, int wide, int64_t i) { return wide ? ((const int64_t *)ids)[i] : ((const int32_t *)ids)[i]; }

// The rows of a tile by adapter: list[start[s]] .. list[start[s + 1] - 1] are those of the s-th adapter that occurs (-1: none, -2: an id outside the bank)
struct alignas(16) RowGroups {
    int id_of_row[LR_ROWS], size[LR_ROWS];         // size: of the group that a row is the first of, else 0
    int list[LR_ROWS], start[LR_ROWS + 1], id[LR_ROWS], groups;
};
__device__ __forceinline__ void group_rows(const LowRankParams &p, int row0, RowGroups &g) {
    const int tid = threadIdx.x, n = min(LR_ROWS, p.M - row0);
    int mine = INT32_MIN;                // rows behind the last form a group of their own, the last one
    if (tid < n) {
        const int64_t id = id_at(p.ids, p.wide_ids, row0 + tid);
        mine = id == -1 ? -1 : id < 0 || id >= p.n_adapters ? -2 : (int)id;
    }
    if (tid < LR_ROWS) g.id_of_row[tid] = mine;
    __syncthreads();
    const bool same = __syncthreads_and(tid >= n || mine == g.id_of_row[0]);
    if (same) {                          // the usual case of a long chunk
        if (tid < n) g.list[tid] = tid;
        if (tid == 0) { g.start[0] = 0; g.start[1] = n; g.id[0] = mine; g.groups = 1; }
        __syncthreads();
        return;
    }
    uint64_t equal = 0;                  // the rows of this row's adapter
    if (tid < LR_ROWS) {
#pragma unroll
        for (int j = 0; j < LR_ROWS; j += 4) {
            const int4 v = *(const int4 *)(g.id_of_row + j);
            equal |= (uint64_t)((v.x == mine) | (v.y == mine) << 1 | (v.z == mine) << 2 | (v.w == mine) << 3) << j;
        }
        g.size[tid] = __ffsll(equal) - 1 == tid ? __popcll(equal) : 0;
    }
    __syncthreads();
    if (tid < LR_ROWS) {
        const int f = __ffsll(equal) - 1;
        int before = 0, group = 0;       // rows and groups whose first row stands in front of this group's
#pragma unroll
        for (int j = 0; j < LR_ROWS; j += 4) {
            const int4 v = *(const int4 *)(g.size + j);
            before += (j < f ? v.x : 0) + (j + 1 < f ? v.y : 0) + (j + 2 < f ? v.z : 0) + (j + 3 < f ? v.w : 0);
            group += (j < f && v.x) + (j + 1 < f && v.y) + (j + 2 < f && v.z) + (j + 3 < f && v.w);
        }
        if (tid < n) {
            const int place = before + __popcll(equal & (((uint64_t)1 << tid) - 1));
            g.list[place] = tid;
            if (f == tid) { g.start[group] = place; g.id[group] = mine; }
            if (place == n - 1) { g.start[group + 1] = n; g.groups = group + 1; }
        }
    }
    __syncthreads();
}

// The sums over part blockIdx.x of K of a tile's inner products.  Ranks on M, rows on N.  A warp takes 16 rows and 16 MT ranks at a time; warps that are not needed for rows share the steps
// of 32 k, and their sums are added in order through shared memory.  Lanes without a row or a rank read another's: what they compute is not looked at, and no load waits behind a branch.
template <int MT>
__global__ void __launch_bounds__(LR_THREADS) low_rank_inner_kernel(const __grid_constant__ LowRankParams p) {
    __shared__ RowGroups groups;
    constexpr int PITCH = MT * 16 + 4;
    __shared__ float red[LR_WARPS][16][PITCH];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4;
    const int row0 = blockIdx.y * LR_ROWS, steps = p.K / 32, per_shard = (p.rank + 15) / 16, tiles = p.n_shards * per_shard;
    const int step0 = (int)((int64_t)blockIdx.x * steps / p.parts), step1 = (int)((int64_t)(blockIdx.x + 1) * steps / p.parts);
    pdl_wait();
    pdl_trigger();
    group_rows(p, row0, groups);
    for (int s = blockIdx.z; s < groups.groups; s += gridDim.z) {
        const int id = groups.id[s], at = groups.start[s], count = groups.start[s + 1] - at;
        if (id < 0) continue;
        const int row_warps = count <= 16 ? 1 : count <= 32 ? 2 : 4, k_warps = LR_WARPS / row_warps, rw = warp % row_warps, kw = warp / row_warps;
        const __nv_bfloat16 *x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = rw * 16 + j * 8 + g;
            x[j] = p.x + (int64_t)(row0 + groups.list[at + min(r, count - 1)]) * p.ldx + t * 8;
        }
        for (int tile0 = 0; tile0 < tiles; tile0 += MT) {
            const __nv_bfloat16 *a[MT][2];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int tile = min(tile0 + i, tiles - 1), shard = tile / per_shard, r = min((tile - shard * per_shard) * 16 + j * 8 + g, p.rank - 1);
                    a[i][j] = p.a + ((int64_t)id * p.n_shards * p.rank + shard * p.rank + r) * p.K + t * 8;
                }
            float acc[MT][2][4] = {};
#pragma unroll 2
            for (int step = step0 + kw; step < step1; step += k_warps) {
                uint4 xv[2], av[MT][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) xv[j] = *(const uint4 *)(x[j] + step * 32);
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) av[i][j] = *(const uint4 *)(a[i][j] + step * 32);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uint32_t lo[4] = {av[i][0].x, av[i][1].x, av[i][0].y, av[i][1].y}, hi[4] = {av[i][0].z, av[i][1].z, av[i][0].w, av[i][1].w};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_bf16(acc[i][j], lo, xv[j].x, xv[j].y);
                        mma_bf16(acc[i][j], hi, xv[j].z, xv[j].w);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) red[warp][j * 8 + t * 2 + (e & 1)][i * 16 + g + (e >> 1) * 8] = acc[i][j][e];
            __syncthreads();
            for (int i = tid; i < count * MT * 16; i += LR_THREADS) {
                const int r = i / (MT * 16), c = i - r * (MT * 16), tile = tile0 + c / 16;
                if (tile >= tiles) continue;
                float sum = 0.0f;
                for (int k = 0; k < k_warps; ++k) sum += red[k * row_warps + r / 16][r % 16][c];
                const int shard = tile / per_shard, rank = (tile - shard * per_shard) * 16 + c % 16;
                p.inner[((int64_t)blockIdx.x * p.M + row0 + groups.list[at + r]) * (p.n_shards * p.ranks) + shard * p.ranks + rank] = sum * p.scales[id * p.n_shards + shard];
            }
            __syncthreads();
        }
    }
}

// base + B (A x) in `cols` columns of one shard.  Rows on M, columns on N; the inner values enter as two bf16 parts (the value and what its rounding left: one part would add an error as
// large as the output's rounding).  A warp takes 32 columns, whose order over its four MMAs gives a lane eight neighbours: base and out move 16 bytes at a time.
template <int KS>
__global__ void __launch_bounds__(LR_THREADS) low_rank_outer_kernel(const __grid_constant__ LowRankParams p) {
    constexpr int R = KS * 16, PITCH = R + 8;
    __shared__ RowGroups groups;
    __shared__ __align__(16) __nv_bfloat16 big[LR_ROWS][PITCH], small[LR_ROWS][PITCH];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4, row0 = blockIdx.y * LR_ROWS;
    int shard = 0;
    int64_t block = blockIdx.x;
    while (true) {                       // which shard's columns
        const int64_t n = (p.edges[shard + 1] - p.edges[shard] + p.cols - 1) / p.cols;
        if (block < n) break;
        block -= n;
        ++shard;
    }
    const int64_t col0 = p.edges[shard] + block * p.cols;
    const int ncols = (int)min((int64_t)p.cols, p.edges[shard + 1] - col0);
    const bool vec = p.vec && ncols >= 8;
    pdl_wait();
    pdl_trigger();
    group_rows(p, row0, groups);
    for (int s = blockIdx.z; s < groups.groups; s += gridDim.z) {
        const int id = groups.id[s], at = groups.start[s], count = groups.start[s + 1] - at;
        if (id < 0) {
            if (id == -2 && blockIdx.x == 0 && tid == 0) atomicMax(p.status, GQ_DEV_BAD_SHAPE);
            if (id == -2 || p.out != p.base)
                for (int i = tid; i < count * ncols; i += LR_THREADS) {
                    const int64_t m = row0 + groups.list[at + i / ncols], n = col0 + i % ncols;
                    p.out[m * p.ld_out + n] = id == -2 ? __ushort_as_bfloat16(0x7fc0) : p.base[m * p.ld_base + n];
                }
            continue;
        }
        for (int i = tid; i < (count + 15) / 16 * 16 * R; i += LR_THREADS) {
            const int r = i / R, k = i % R;
            float v = 0.0f;
            if (r < count && k < p.rank) {
                const float *src = p.inner + (int64_t)(row0 + groups.list[at + r]) * (p.n_shards * p.ranks) + shard * p.ranks + k;
                for (int part = 0; part < p.parts; ++part) v += src[(int64_t)part * p.M * (p.n_shards * p.ranks)];
            }
            const __nv_bfloat16 b = __float2bfloat16_rn(v);
            big[r][k] = b;
            small[r][k] = __float2bfloat16_rn(v - __bfloat162float(b));
        }
        __syncthreads();
        for (int n0 = warp * 32; n0 < ncols; n0 += LR_WARPS * 32) {
            uint32_t bf[4][KS][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = n0 + 8 * (g / 2) + 2 * i + (g & 1);
                const __nv_bfloat16 *src = p.b + ((int64_t)id * p.n_total + col0 + min(n, ncols - 1)) * p.rank;
                if constexpr (KS == 1) {
                    const bool in = t * 4 < p.rank;            // ranks that only fill the tile are zero here and in the inner values
                    const uint2 v = *(const uint2 *)(src + (in ? t * 4 : 0));
                    bf[i][0][0] = in ? v.x : 0u; bf[i][0][1] = in ? v.y : 0u;
                } else {
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        const bool in = k * 16 + t * 8 < p.rank;
                        const uint4 v = *(const uint4 *)(src + (in ? k * 16 + t * 8 : 0));
                        bf[i][k][0] = in ? v.x : 0u; bf[i][k][1] = in ? v.y : 0u; bf[i][k + 1][0] = in ? v.z : 0u; bf[i][k + 1][1] = in ? v.w : 0u;
                    }
                }
            }
            for (int m0 = 0; m0 < count; m0 += 16) {
                const int n = n0 + t * 8;
                const bool have[2] = {m0 + g < count && n < ncols, m0 + g + 8 < count && n < ncols}, whole = n + 8 <= ncols;
                int64_t m[2];
                uint4 old[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) m[j] = row0 + groups.list[at + min(m0 + g + 8 * j, count - 1)];
                if (vec) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) old[j] = *(const uint4 *)(p.base + m[j] * p.ld_base + col0 + (whole ? n : 0));       // of an eighth that ends early: below
                }
                if (!vec || !whole)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const __nv_bfloat16 *src = p.base + m[j] * p.ld_base + col0;
                        uint16_t e[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) e[x] = __bfloat16_as_ushort(src[min(n + x, ncols - 1)]);
                        memcpy(&old[j], e, 16);
                    }
                float acc[4][4] = {};
#pragma unroll
                for (int k = 0; k < KS; k += KS == 1 ? 1 : 2) {
                    uint32_t hi[2][4], lo[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int r = m0 + g + 8 * j;
                        if constexpr (KS == 1) {
                            const uint2 v = *(const uint2 *)&big[r][t * 4], w = *(const uint2 *)&small[r][t * 4];
                            hi[0][j] = v.x; hi[0][j + 2] = v.y;
                            lo[0][j] = w.x; lo[0][j + 2] = w.y;
                        } else {
                            const uint4 v = *(const uint4 *)&big[r][k * 16 + t * 8], w = *(const uint4 *)&small[r][k * 16 + t * 8];
                            hi[0][j] = v.x; hi[0][j + 2] = v.y; hi[1][j] = v.z; hi[1][j + 2] = v.w;
                            lo[0][j] = w.x; lo[0][j + 2] = w.y; lo[1][j] = w.z; lo[1][j + 2] = w.w;
                        }
                    }
#pragma unroll
                    for (int q = 0; q < (KS == 1 ? 1 : 2); ++q)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_bf16(acc[i], hi[q], bf[i][k + q][0], bf[i][k + q][1]);
                            mma_bf16(acc[i], lo[q], bf[i][k + q][0], bf[i][k + q][1]);
                        }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (!have[j]) continue;
                    const uint32_t w[4] = {old[j].x, old[j].y, old[j].z, old[j].w};
                    uint32_t y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = bf16_pair(__uint_as_float(w[i] << 16) + acc[i][2 * j], __uint_as_float(w[i] & 0xffff0000u) + acc[i][2 * j + 1]);
                    __nv_bfloat16 *dst = p.out + m[j] * p.ld_out + col0 + n;
                    if (vec && whole) *(uint4 *)dst = make_uint4(y[0], y[1], y[2], y[3]);
                    else {
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (n + x < ncols) dst[x] = __ushort_as_bfloat16((uint16_t)(y[x / 2] >> (16 * (x & 1))));
                    }
                }
            }
        }
        __syncthreads();
    }
}

}  // namespace gq
