// Low-rank adapters beside a shared projection: out = base + scale * B (A x) for each row's own adapter.
//
// Two launches: the inner products A x (K split over the blocks of a cluster, their sums left in the workspace as two bf16 parts) and the outer products B (A x) with the addition.  No row's sums
// ever hold another adapter's numbers, and rows of one adapter need not stand together: the inner products sort a tile's 64 rows by adapter and multiply each adapter's own; the outer ones multiply
// a tile of 16 rows (or 4) once for every adapter in it and keep that one's rows.  In decode both read bf16 operands from global memory straight into the fragments of mma.sync m16n8k16: any order
// of k serves as long as both operands have the same, so a lane takes 8 neighbours (16 bytes) where the instruction names scattered ones.  In chunks of prompts both go through shared memory.
// Bound by bytes, in decode those of the adapters (below a few MB latency is all), in chunks those of base and out.
//
// Measured (graph of calls): one row beside qkv, rank 16, 6.2 us (two launches, two rounds of memory, a cluster's sums); 27 rows of 8 adapters of rank 32 beside gate_up 11.8 (18 MB, floor 2.8); 64 rows of 16
// of rank 64 beside down 24 (49 MB, floor 7.6; 37 where A is not in the L2): the inner warps go through four or five whole latencies one behind the other, two barriers of the cluster for every adapter, at 15 % of DRAM's rate, and the outer
// tiles of 4 rows load one adapter's columns behind another's; 2,051 rows of rank 16 beside gate_up 83 (312 MB, floor 48), of
// rank 128 beside qkv 95 (floor 16): there the inner products run at 160 TFLOP/s, and mma.sync of 64 x 64 tiles is what bounds them.
// Tried: all of a block's part of A asked of the L2 at once (m64 36 to 36 us, one row 6.2 to 6.5); sums of the parts by the outer blocks (m64 7 us less in the inner, 8 more in the outer kernel); decode through the chunk kernels (m64 24 to 36); the base straight to registers with two to
// four tiles ahead (m2051 outer 86 to 110); 64 rows x 256 or 32 x 512 columns in shared memory with two blocks to an SM (79 and 77 against 67 with four blocks of 32 x 256).
#pragma once
#include "gq_bf16.cuh"

namespace gq {

constexpr int LR_ROWS = 64, LR_THREADS = 256, LR_WARPS = LR_THREADS / 32;

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

struct LowRankParams {
    const __nv_bfloat16 *base, *x, *a, *b;
    const float *scales;
    const void *ids;
    __nv_bfloat16 *out;
    __nv_bfloat16 *big, *small;  // workspace: the scaled inner values [M, n_shards * ranks] as bf16, and what that rounding left
    int *status;
    int64_t ld_base, ldx, ld_out, n_total;
    int64_t edges[9];            // first column of each shard, and the end
    int M, K, n_shards, n_adapters, rank, ranks, parts, wide_ids;       // ranks: the rank as the outer products see it, 16, 32, 64 or 128
    int group_blocks;            // blocks along z that share a tile's adapters; the others take further ranks
    int vec;                     // base and out can be read and written 16 bytes at a time
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

// The sums of `count` rows and RANKS ranks, `of(row, rank)` in every block's shared memory, over the blocks of the cluster in order -> the workspace
template <int RANKS, class OF> __device__ __forceinline__ void store_inner(const LowRankParams &p, const RowGroups &groups, int at, int count, int id, int row0, int tile0, OF of) {
    const int per_shard = (p.rank + 15) / 16, tiles = p.n_shards * per_shard;
    if (p.parts > 1) cluster_sync_all();
    else __syncthreads();
    for (int i = threadIdx.x + blockIdx.x * LR_THREADS; i < count * RANKS; i += LR_THREADS * p.parts) {
        const int r = i / RANKS, c = i - r * RANKS, tile = tile0 + c / 16;
        if (tile >= tiles) continue;
        float sum = 0.0f;
        if (p.parts > 1) {
            const uint32_t from = smem_u32(of(r, c));
            for (int k0 = 0; k0 < p.parts; k0 += 8) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = k0 + k < p.parts ? ld_cluster_f32(map_to_rank(from, k0 + k)) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += v[k];
            }
        } else sum = *of(r, c);
        const int shard = tile / per_shard, rank = (tile - shard * per_shard) * 16 + c % 16;
        sum *= p.scales[id * p.n_shards + shard];
        const int64_t to = (int64_t)(row0 + groups.list[at + r]) * (p.n_shards * p.ranks) + shard * p.ranks + rank;
        // an infinity has nothing left over (inf - inf would make NaN of it), and a finite sum beyond bf16's range is its largest value and a rest
        constexpr float TOP = 3.3895313892515355e38f;
        const bool infinite = isinf(sum);
        const __nv_bfloat16 big = __float2bfloat16_rn(!infinite && fabsf(sum) > TOP ? copysignf(TOP, sum) : sum);
        p.big[to] = big;
        p.small[to] = infinite ? __float2bfloat16_rn(0.0f) : __float2bfloat16_rn(sum - __bfloat162float(big));
    }
    if (p.parts > 1) cluster_sync_all();            // nobody reads this block's sums any more
    else __syncthreads();
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
    const int step0 = (int)((int64_t)blockIdx.x * (steps / 2) / p.parts) * 2, step1 = (int)((int64_t)(blockIdx.x + 1) * (steps / 2) / p.parts) * 2;      // pairs
    pdl_wait();
    pdl_trigger();
    group_rows(p, row0, groups);
    const int tile0 = blockIdx.z / p.group_blocks * MT;            // this block's ranks, in sixteens over all shards
    for (int s = blockIdx.z % p.group_blocks; s < groups.groups; s += p.group_blocks) {
        const int id = groups.id[s], at = groups.start[s], count = groups.start[s + 1] - at;
        if (id < 0) continue;
        const int row_warps = count <= 16 ? 1 : count <= 32 ? 2 : 4, k_warps = LR_WARPS / row_warps, rw = warp % row_warps, kw = warp / row_warps;
        const __nv_bfloat16 *x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = rw * 16 + j * 8 + g;
            x[j] = p.x + (int64_t)(row0 + groups.list[at + min(r, count - 1)]) * p.ldx + t * 8;
        }
        const __nv_bfloat16 *a[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int tile = min(tile0 + i, tiles - 1), shard = tile / per_shard, r = min((tile - shard * per_shard) * 16 + j * 8 + g, p.rank - 1);
                a[i][j] = p.a + ((int64_t)id * p.n_shards * p.rank + shard * p.rank + r) * p.K + t * 8;
            }
        float acc[MT][2][4] = {};
        // two steps at a time, the 128 bytes of a row that lie side by side
#pragma unroll(MT <= 2 ? 2 : 1)
        for (int step = step0 + 2 * kw; step < step1; step += 2 * k_warps) {
            uint4 xv[2][2], av[2][MT][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < 2; ++j) xv[h][j] = *(const uint4 *)(x[j] + (step + h) * 32);
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) av[h][i][j] = *(const uint4 *)(a[i][j] + (step + h) * 32);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uint4 a0 = av[h][i][0], a1 = av[h][i][1];
                    const uint32_t lo[4] = {a0.x, a1.x, a0.y, a1.y}, hi[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_bf16(acc[i][j], lo, xv[h][j].x, xv[h][j].y);
                        mma_bf16(acc[i][j], hi, xv[h][j].z, xv[h][j].w);
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
        // over the warps of this block, then over the blocks of the cluster, both in order
        for (int i = tid; i < count * MT * 16; i += LR_THREADS) {
            const int r = i / (MT * 16), c = i - r * (MT * 16);
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < LR_WARPS; ++k)
                if (k < k_warps) sum += red[k * row_warps + r / 16][r % 16][c];
            red[r / 16][r % 16][c] = sum;              // read by this thread alone so far
        }
        store_inner<MT * 16>(p, groups, at, count, id, row0, tile0, [&](int r, int c) { return &red[r / 16][r % 16][c]; });
    }
}

// The same for chunks, where a tile's rows mostly share an adapter and A is read by many: 64 rows times RANKS ranks, both through shared memory in steps of 64 k (cp.async, a ring of four;
// rows at a pitch of 144 bytes, so that ldmatrix meets no bank twice).  Rows on M; a warp has 16 rows and half of the ranks.
template <int RANKS> struct InnerShape {
    static constexpr int PITCH = 144, STAGES = 4, STAGE = (LR_ROWS + RANKS) * PITCH, SMEM = STAGES * STAGE, RED = RANKS + 4;
    static_assert(LR_ROWS * RED * 4 <= SMEM, "the sums take the ring's place");
};
template <int RANKS>
__global__ void __launch_bounds__(LR_THREADS) low_rank_inner_chunk_kernel(const __grid_constant__ LowRankParams p) {
    using Shape = InnerShape<RANKS>;
    constexpr int PITCH = Shape::PITCH, S = Shape::STAGES, NT = RANKS / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RowGroups groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4, rw = warp % 4, cw = warp / 4;
    const int row0 = blockIdx.y * LR_ROWS, blocks = p.K / 64, per_shard = (p.rank + 15) / 16, tiles = p.n_shards * per_shard, tile0 = blockIdx.z / p.group_blocks * (RANKS / 16);
    const int k0 = (int)((int64_t)blockIdx.x * blocks / p.parts), k1 = (int)((int64_t)(blockIdx.x + 1) * blocks / p.parts);
    pdl_wait();
    pdl_trigger();
    group_rows(p, row0, groups);
    float(*red)[Shape::RED] = (float(*)[Shape::RED])smem;
    for (int s = blockIdx.z % p.group_blocks; s < groups.groups; s += p.group_blocks) {
        const int id = groups.id[s], at = groups.start[s], count = groups.start[s + 1] - at;
        if (id < 0) continue;
        // 16 bytes of a row or rank at a time: 8 threads to a row; rows and ranks that are not there are read as the last
        const __nv_bfloat16 *src[2 + RANKS / 32];
#pragma unroll
        for (int j = 0; j < 2 + RANKS / 32; ++j) {
            const int r = tid / 8 + 32 * (j & 1), c = (tid & 7) * 8;
            if (j < 2) src[j] = p.x + (int64_t)(row0 + groups.list[at + min(r, count - 1)]) * p.ldx + c;
            else {
                const int q = tid / 8 + 32 * (j - 2), tile = min(tile0 + q / 16, tiles - 1), shard = tile / per_shard, rank = min((tile - shard * per_shard) * 16 + q % 16, p.rank - 1);
                src[j] = p.a + ((int64_t)id * p.n_shards * p.rank + shard * p.rank + rank) * p.K + c;
            }
        }
        auto ask = [&](int k) {
            if (k < k1) {
                const uint32_t to = smem_u32(smem) + (k - k0) % S * Shape::STAGE + tid / 8 * PITCH + (tid & 7) * 16;
#pragma unroll
                for (int j = 0; j < 2 + RANKS / 32; ++j) cp_async16(to + j * 32 * PITCH, src[j] + k * 64);
            }
            cp_async_commit();
        };
        for (int i = 0; i < S - 1; ++i) ask(k0 + i);
        float acc[NT][4] = {};
        for (int k = k0; k < k1; ++k) {
            cp_async_wait<S - 2>();
            __syncthreads();
            ask(k + S - 1);
            const uint32_t stage = smem_u32(smem) + (k - k0) % S * Shape::STAGE;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                uint32_t xf[4];
                ldsm4(xf, stage + (rw * 16 + (lane & 15)) * PITCH + h * 32 + (lane >> 4) * 16);
#pragma unroll
                for (int i = 0; i < NT; i += 2) {
                    uint32_t af[4];
                    ldsm4(af, stage + (LR_ROWS + cw * (RANKS / 2) + i * 8 + (lane >> 4) * 8 + (lane & 7)) * PITCH + h * 32 + ((lane >> 3) & 1) * 16);
                    mma_bf16(acc[i], xf, af[0], af[1]);
                    mma_bf16(acc[i + 1], xf, af[2], af[3]);
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[rw * 16 + g + (e >> 1) * 8][cw * (RANKS / 2) + i * 8 + t * 2 + (e & 1)] = acc[i][e];
        store_inner<RANKS>(p, groups, at, count, id, row0, tile0, [&](int r, int c) { return &red[r][c]; });
    }
}

// base + B (A x), the outer products.  Rows on M, columns on N; the inner values enter as two bf16 parts (the value and what its rounding left: one part would add an error as large as the
// output's rounding).  A warp takes 32 columns, whose order over its four MMAs gives a lane eight neighbours, so that base and out move 16 bytes at a time; the base is what the accumulators
// start from.  A tile of 16 rows that has several adapters is multiplied once with each and keeps that one's rows.

// a warp's 32 columns of adapter `id` as B operands: of shard columns n0 .. of which `here` are real
template <int KS> __device__ __forceinline__ void load_columns(const LowRankParams &p, int id, int64_t col, int here, int lane, uint32_t (&bf)[4][KS][2]) {
    const int g = lane / 4, t = lane % 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat16 *src = p.b + ((int64_t)id * p.n_total + col + min(8 * (g / 2) + 2 * i + (g & 1), here - 1)) * p.rank;
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
}
// rows g and g + 8 of the inner values (big and small: where they start) times the columns, onto acc
template <int KS, class B, class S> __device__ __forceinline__ void add_products(const LowRankParams &p, B big, S small, const uint32_t (&bf)[4][KS][2], int t, float (&acc)[4][4]) {
#pragma unroll
    for (int k = 0; k < KS; k += KS == 1 ? 1 : 2) {
        uint32_t hi[2][4], lo[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (KS == 1) {
                const bool in = t * 4 < p.rank;
                const uint2 v = *(const uint2 *)(big(j) + t * 4), x = *(const uint2 *)(small(j) + t * 4);
                hi[0][j] = in ? v.x : 0u; hi[0][j + 2] = in ? v.y : 0u;
                lo[0][j] = in ? x.x : 0u; lo[0][j + 2] = in ? x.y : 0u;
            } else {
                const bool in = k * 16 + t * 8 < p.rank;
                const uint4 v = *(const uint4 *)(big(j) + k * 16 + t * 8), x = *(const uint4 *)(small(j) + k * 16 + t * 8);
                hi[0][j] = in ? v.x : 0u; hi[0][j + 2] = in ? v.y : 0u; hi[1][j] = in ? v.z : 0u; hi[1][j + 2] = in ? v.w : 0u;
                lo[0][j] = in ? x.x : 0u; lo[0][j + 2] = in ? x.y : 0u; lo[1][j] = in ? x.z : 0u; lo[1][j + 2] = in ? x.w : 0u;
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
}
__device__ __forceinline__ int adapter_of(const LowRankParams &p, int row) {
    const int64_t id = id_at(p.ids, p.wide_ids, row);
    return id == -1 ? -1 : id < 0 || id >= p.n_adapters ? -2 : (int)id;
}
// eight bf16 values of two rows -> accumulators (columns 8 t + 2 i and the next: of row g in 0, 1, of row g + 8 in 2, 3), and back
__device__ __forceinline__ void unpack_rows(const uint4 (&w)[2], float (&res)[4][4]) {
    const uint32_t u[2][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w}};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) { res[i][2 * j] = __uint_as_float(u[j][i] << 16); res[i][2 * j + 1] = __uint_as_float(u[j][i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack_row(const float (&res)[4][4], int j) {
    return make_uint4(bf16_pair(res[0][2 * j], res[0][2 * j + 1]), bf16_pair(res[1][2 * j], res[1][2 * j + 1]), bf16_pair(res[2][2 * j], res[2][2 * j + 1]),
                      bf16_pair(res[3][2 * j], res[3][2 * j + 1]));
}
// one tile of rows: `mine` is the adapter of row lane & 15, `have` the one whose columns bf holds
template <int KS, class B, class S> __device__ __forceinline__ void outer_tile(const LowRankParams &p, int mine, int &have, uint32_t (&bf)[4][KS][2], int64_t col, int here, int lane, B big, S small,
                                                                               float (&res)[4][4], int (&of_row)[2]) {
    const int g = lane / 4, t = lane % 4;
    of_row[0] = __shfl_sync(~0u, mine, g);
    of_row[1] = __shfl_sync(~0u, mine, g + 8);
    uint32_t todo = __ballot_sync(~0u, mine >= 0) & 0xffffu;
    while (todo) {
        const int of = __shfl_sync(~0u, mine, __ffs(todo) - 1);
        const uint32_t its = __ballot_sync(~0u, mine == of) & 0xffffu;
        todo &= ~its;
        if (of != have) {
            have = of;
            load_columns<KS>(p, of, col, here, lane, bf);
        }
        if (its == 0xffffu) {
            add_products<KS>(p, big, small, bf, t, res);
            return;
        }
        float acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = res[i][j];
        add_products<KS>(p, big, small, bf, t, acc);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) res[i][j] = of_row[j >> 1] == of ? acc[i][j] : res[i][j];
    }
    if (__any_sync(~0u, mine == -2)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (of_row[j >> 1] == -2)
#pragma unroll
                for (int i = 0; i < 4; ++i) res[i][j] = __int_as_float(0x7fc00000);
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicMax(p.status, GQ_DEV_BAD_SHAPE);
    }
}
// which shard's columns block `block` of `cols` has: first of them, and how many
__device__ __forceinline__ int shard_of(const LowRankParams &p, int64_t block, int cols, int64_t &col0, int &ncols) {
    int shard = 0;
    while (true) {
        const int64_t n = (p.edges[shard + 1] - p.edges[shard] + cols - 1) / cols;
        if (block < n) break;
        block -= n;
        ++shard;
    }
    col0 = p.edges[shard] + block * cols;
    ncols = (int)min((int64_t)cols, p.edges[shard + 1] - col0);
    return shard;
}

// Decode: a warp by itself has 32 columns of TILE rows.  Where every row may have an adapter of its own TILE is 4 (the MMA's other rows idle, but no more than four adapters stand one behind
// the other), with a small bank 16.
constexpr int LR_OUTER_WARPS = 4;
template <int KS, int TILE>
__global__ void __launch_bounds__(LR_OUTER_WARPS * 32) low_rank_few_kernel(const __grid_constant__ LowRankParams p) {
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane % 4, row0 = blockIdx.y * TILE, last = min(row0 + TILE, p.M) - 1;
    int64_t col0;
    int ncols;
    const int shard = shard_of(p, blockIdx.x, LR_OUTER_WARPS * 32, col0, ncols);
    col0 += threadIdx.x / 32 * 32;
    ncols = min(ncols - (int)(threadIdx.x / 32) * 32, 32);
    const int n = t * 8;
    const bool full = p.vec && n + 8 <= ncols;                     // this lane's columns: 16 aligned bytes
    pdl_wait();
    pdl_trigger();
    if (ncols <= 0) return;
    const int mine = adapter_of(p, min(row0 + (lane & 15), last));
    constexpr int HALVES = TILE > 8 ? 2 : 1;                       // rows g, and g + 8
    uint4 w[2] = {};
    int64_t at[2] = {};
#pragma unroll
    for (int j = 0; j < HALVES; ++j) {
        const int64_t row = min(row0 + g + 8 * j, last);
        const __nv_bfloat16 *src = p.base + row * p.ld_base + col0 + n;
        at[j] = row * (p.n_shards * p.ranks) + shard * p.ranks;
        if (full) w[j] = *(const uint4 *)src;
        else {
            uint16_t e[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) e[x] = n + x < ncols ? __bfloat16_as_ushort(src[x]) : 0;
            memcpy(&w[j], e, 16);
        }
    }
    if (HALVES == 1) at[1] = at[0];
    float res[4][4];
    unpack_rows(w, res);
    uint32_t bf[4][KS][2];
    int have = -1, of_row[2];
    outer_tile<KS>(p, mine, have, bf, col0, ncols, lane, [&](int j) { return p.big + at[j]; }, [&](int j) { return p.small + at[j]; }, res, of_row);
#pragma unroll
    for (int j = 0; j < HALVES; ++j) {
        if (row0 + g + 8 * j > last || (of_row[j] == -1 && p.out == p.base)) continue;         // in place, rows without an adapter stay as they are
        const uint4 y = pack_row(res, j);
        __nv_bfloat16 *dst = p.out + (row0 + g + 8 * j) * p.ld_out + col0 + n;
        if (full) *(uint4 *)dst = y;
        else {
            uint16_t e[8];
            memcpy(e, &y, 16);
#pragma unroll
            for (int x = 0; x < 8; ++x)
                if (n + x < ncols) dst[x] = __ushort_as_bfloat16(e[x]);
        }
    }
}

// Chunks: a block keeps its 256 columns and walks down the rows, 32 at a time, so an adapter's part of B is read once.  Base and inner values come through shared memory, a tile ahead, and the
// sums leave from there in whole lines: what is in flight does not depend on registers, and a thread's addresses only step.
template <int KS> struct ChunkShape {
    static constexpr int COLS = 256, ROWS = 32, PITCH = COLS * 2 + 64, BLOCKS = KS == 1 ? 4 : KS == 2 ? 3 : 2;        // rows g and g + 1 in different banks; blocks to an SM
    static constexpr int RP = KS * 16 + 8, STAGE = ROWS * PITCH + 2 * ROWS * RP * 2, SMEM = 2 * STAGE;
};
template <int KS>
__global__ void __launch_bounds__(LR_THREADS, ChunkShape<KS>::BLOCKS) low_rank_chunk_kernel(const __grid_constant__ LowRankParams p, int tiles) {
    using Shape = ChunkShape<KS>;
    constexpr int COLS = Shape::COLS, ROWS = Shape::ROWS, PITCH = Shape::PITCH, RP = Shape::RP, E = COLS / 8, STEP = LR_THREADS / E, R8 = KS * 2;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4;
    int64_t col0;
    int ncols;
    const int shard = shard_of(p, blockIdx.x, COLS, col0, ncols);
    const int row0 = blockIdx.y * tiles * ROWS, row1 = min(row0 + tiles * ROWS, p.M), eighths = p.vec ? ncols / 8 : 0, rest = ncols - eighths * 8;
    const int er = tid / E, ec = tid % E;                          // this thread's row and eighth of a tile's copies
    pdl_wait();
    pdl_trigger();
    if (row0 >= row1) return;
    auto ask = [&](int row, int stage) {
        if (row < row1) {
            uint8_t *to = smem + stage * Shape::STAGE;
            const int rows = min(ROWS, row1 - row);
            if (ec < eighths) {
                const __nv_bfloat16 *src = p.base + (row + er) * p.ld_base + col0 + ec * 8;
                const uint32_t dst = smem_u32(to) + er * PITCH + ec * 16;
#pragma unroll
                for (int i = 0; i < ROWS / STEP; ++i, src += STEP * p.ld_base)
                    if (er + i * STEP < rows) cp_async16(dst + i * STEP * PITCH, src);
            }
            for (int i = tid; i < rows * rest; i += LR_THREADS) {  // columns that do not fill 16 aligned bytes
                const int r = i / rest, c = eighths * 8 + i % rest;
                *(__nv_bfloat16 *)(to + r * PITCH + c * 2) = p.base[(row + r) * p.ld_base + col0 + c];
            }
            for (int i = tid; i < rows * R8 * 2; i += LR_THREADS) {        // the workspace's rows are `ranks` long
                const int small = i >= rows * R8, x = i - small * rows * R8, r = x / R8, c = x % R8;
                const __nv_bfloat16 *src = (small ? p.small : p.big) + (int64_t)(row + r) * (p.n_shards * p.ranks) + shard * p.ranks + c * 8;
                cp_async16(smem_u32(to + ROWS * PITCH + (small * ROWS + r) * RP * 2 + c * 16), src);
            }
        }
        cp_async_commit();
    };
    uint32_t bf[4][KS][2];
    int have = -1;
    const int n0 = warp * 32;
    ask(row0, 0);
    for (int row = row0, stage = 0; row < row1; row += ROWS, stage ^= 1) {
        ask(row + ROWS, stage ^ 1);
        int mine[ROWS / 16];
#pragma unroll
        for (int i = 0; i < ROWS / 16; ++i) mine[i] = adapter_of(p, min(row + i * 16 + (lane & 15), row1 - 1));
        cp_async_wait<1>();
        __syncthreads();
        uint8_t *base = smem + stage * Shape::STAGE;
        const __nv_bfloat16 *big = (const __nv_bfloat16 *)(base + ROWS * PITCH), *small = big + ROWS * RP;
        if (n0 < ncols)
#pragma unroll
            for (int i = 0; i < ROWS / 16; ++i) {
                if (row + i * 16 >= row1) continue;
                uint4 *at[2], w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    at[j] = (uint4 *)(base + (i * 16 + g + 8 * j) * PITCH + (n0 + t * 8) * 2);
                    w[j] = *at[j];
                }
                float res[4][4];
                int of_row[2];
                unpack_rows(w, res);
                auto of = [&](const __nv_bfloat16 *v) { return [=](int j) { return v + (i * 16 + g + 8 * j) * RP; }; };
                outer_tile<KS>(p, mine[i], have, bf, col0 + n0, min(ncols - n0, 32), lane, of(big), of(small), res, of_row);
                *at[0] = pack_row(res, 0);
                *at[1] = pack_row(res, 1);
            }
        __syncthreads();
        const int rows = min(ROWS, row1 - row);
        const bool keep = p.out == p.base;                         // in place, rows without an adapter stay as they are
        if (ec < eighths) {
            __nv_bfloat16 *dst = p.out + (row + er) * p.ld_out + col0 + ec * 8;
            const uint8_t *src = base + er * PITCH + ec * 16;
#pragma unroll
            for (int i = 0; i < ROWS / STEP; ++i, dst += STEP * p.ld_out)
                if (er + i * STEP < rows && !(keep && adapter_of(p, row + er + i * STEP) == -1)) *(uint4 *)dst = *(const uint4 *)(src + i * STEP * PITCH);
        }
        for (int i = tid; i < rows * rest; i += LR_THREADS) {
            const int r = i / rest, c = eighths * 8 + i % rest;
            if (!(keep && adapter_of(p, row + r) == -1)) p.out[(row + r) * p.ld_out + col0 + c] = *(const __nv_bfloat16 *)(base + r * PITCH + c * 2);
        }
        __syncthreads();                                           // the next request writes here
    }
}

}  // namespace gq
