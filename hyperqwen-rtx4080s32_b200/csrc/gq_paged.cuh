// Attention of a sequence's newest tokens over its keys and values in the pages of a cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c q . k_j - m),  c = scale log2 e,  m the running maximum: one pass over keys and values.
//
// Bound by the bytes of the cache: a key-value head's key and value are 4 head_dim bytes, and the rows that share them (the query heads of the group, times the new tokens)
// are few.  So the work is cut evenly by keys, not by sequences: the units of all (sequence, kv head, tile of rows) in a line, a unit being KG * 16 keys, and block c of G takes
// units [c W / G, (c + 1) W / G).  A segment that lies in one block is finished there; of the others each block leaves its unnormalised rows, maxima and sums
// in the workspace, and join_parts_kernel adds them in block order.  Every block finds its place from lens alone, so the host need not know them, and the order of all sums
// follows from the lengths and the number of SMs.
//
// A block is four warps: RG row groups of 16 rows times KG = 4 / RG key groups.  A key group streams 16 keys at a time through a ring of its own in shared memory (cp.async, 16 bytes, chunks
// exclusive-ored with the row, so that ldmatrix meets no bank twice) and its RG warps multiply them: scores as q k^T (mma.sync m16n8k16, rows on M), the probabilities as they leave the
// accumulators are the A operand of p v.  p enters as two bf16 parts (p and what its rounding left): one part would add an error as large as the output's own rounding, and the tensor pipe has room.
// tcgen05 has nothing to give here: 16 rows of its 128 would be used, and the loads are the bound.
#pragma once
#include "gq_common.cuh"

namespace gq {

constexpr int PA_THREADS = 128, PA_STAGES = 3;

struct PagedParams {
    gq_attention_args a;
    int *status;
    int64_t *first;         // workspace: [n_seqs] first unit of each sequence, then W
    float2 *stats;          // [2 G][rows of a tile]: maximum, sum
    float *parts;           // [2 G][rows of a tile][head_dim]
    int group, blocks;
    float scale2;           // scale * log2 e
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &v, 4);
    return u;
}
// two probabilities as bf16 and what that rounding left, as bf16
__device__ __forceinline__ void bf16_parts(float lo, float hi, uint32_t &big, uint32_t &small) {
    big = bf16_pair(lo, hi);
    small = bf16_pair(lo - __uint_as_float(big << 16), hi - __uint_as_float(big & 0xffff0000u));
}

// A sequence's tokens and keys, and how its rows and keys are cut
struct SeqSpan {
    int64_t tok0;     // its first token
    int n, len;       // new tokens, keys
};
__device__ __forceinline__ SeqSpan seq_span(const gq_attention_args &a, int64_t s) {
    SeqSpan v;
    if (a.q_starts) {
        const int64_t q0 = min(max((int64_t)a.q_starts[s], (int64_t)0), a.T), q1 = min(max((int64_t)a.q_starts[s + 1], q0), a.T);
        v.tok0 = q0; v.n = (int)(q1 - q0);
    } else {
        v.n = (int)(a.T / a.n_seqs); v.tok0 = s * v.n;
    }
    v.len = max(a.lens[s], 0);
    return v;
}
// keys that a tile's last row sees
__device__ __forceinline__ int tile_keys(const SeqSpan &v, int tile, int rows, int group) {
    const int last = min(v.n - 1, (int)(((int64_t)(tile + 1) * rows - 1) / group));
    return max(0, v.len - v.n + last + 1);
}
__device__ __forceinline__ int tiles_of(const SeqSpan &v, int rows, int group) { return (int)(((int64_t)v.n * group + rows - 1) / rows); }
__device__ __forceinline__ int64_t head_units(const SeqSpan &v, int rows, int group, int unit) {
    int64_t u = 0;
    for (int t = 0, n = tiles_of(v, rows, group); t < n; ++t) u += (tile_keys(v, t, rows, group) + unit - 1) / unit;
    return u;
}

// Where a block's walk over the line of units stands: the segment (sequence, kv head, tile) and the next unit in it
struct Cursor {
    int64_t seq;
    SeqSpan v;
    int head, tile, tiles, unit, units, keys;
};
template <int ROWS, int UNIT> __device__ __forceinline__ void load_segment(const PagedParams &p, Cursor &c) {
    c.keys = tile_keys(c.v, c.tile, ROWS, p.group);
    c.units = (c.keys + UNIT - 1) / UNIT;
}
// to the next segment that has units (there is one: the caller counts)
template <int ROWS, int UNIT> __device__ __forceinline__ void next_segment(const PagedParams &p, Cursor &c) {
    c.unit = 0;
    do {
        if (++c.tile >= c.tiles) {
            c.tile = 0;
            if (++c.head == p.a.n_kv_heads || c.tiles == 0) {
                c.head = 0;
                do {
                    if (++c.seq >= p.a.n_seqs) { c.units = 0; return; }
                    c.v = seq_span(p.a, c.seq);
                    c.tiles = tiles_of(c.v, ROWS, p.group);
                } while (c.tiles == 0);
            }
        }
        load_segment<ROWS, UNIT>(p, c);
    } while (c.units == 0);
}

template <int D, int RG> struct PagedShape {
    static constexpr int KG = 4 / RG, ROWS = 16 * RG, UNIT = 16 * KG;
    static constexpr int STAGE = 2 * 16 * D * 2;                                // keys and values of 16 keys, bytes
    static constexpr int RING = KG * PA_STAGES * STAGE, Q = D > 128 ? ROWS * D * 2 : 0, MERGE = KG > 1 ? ROWS * D * 4 : 0;
    static constexpr int SMEM = RING + Q + MERGE + (KG > 1 ? KG * ROWS * 8 : 0) + KG * PA_STAGES * 4 + 128;
};

template <int D, int RG>
__global__ void __launch_bounds__(PA_THREADS) paged_attention_kernel(const __grid_constant__ PagedParams p) {
    using Shape = PagedShape<D, RG>;
    constexpr int KG = Shape::KG, ROWS = Shape::ROWS, UNIT = Shape::UNIT, STAGE = Shape::STAGE, S = PA_STAGES, CH = D / 8, NT = D / 8, KK = D / 16;
    constexpr bool QREG = D <= 128;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *q_sm = smem + Shape::RING;
    float *merge = (float *)(q_sm + Shape::Q);
    float2 *stat_sm = (float2 *)((uint8_t *)merge + Shape::MERGE);
    uint32_t *bad_sm = (uint32_t *)((uint8_t *)stat_sm + (KG > 1 ? KG * ROWS * 8 : 0));
    __shared__ int64_t scan[PA_THREADS / 32], place[3];
    const gq_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, rg = warp % RG, kg = warp / RG, g = lane / 4, t = lane % 4;
    pdl_wait();
    pdl_trigger();

    // ---- this block's units ----
    int64_t total, w0, w1;
    Cursor use;
    {
        const int64_t each = (a.n_seqs + PA_THREADS - 1) / PA_THREADS, s0 = min(tid * each, a.n_seqs), s1 = min(s0 + each, a.n_seqs);
        int64_t mine = 0;
        for (int64_t s = s0; s < s1; ++s) mine += head_units(seq_span(a, s), ROWS, p.group, UNIT) * a.n_kv_heads;
        int64_t upto = mine;
        for (int o = 1; o < 32; o *= 2) {
            const int64_t v = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        total = 0;
        for (int w = 0; w < PA_THREADS / 32; ++w) {
            if (w < warp) upto += scan[w];
            total += scan[w];
        }
        const int64_t blocks = min((int64_t)p.blocks, max(total, (int64_t)1));
        w0 = blockIdx.x < blocks ? blockIdx.x * total / blocks : total;
        w1 = blockIdx.x < blocks ? (blockIdx.x + 1) * total / blocks : total;
        int64_t at = upto - mine;
        if (blockIdx.x == 0 || (w0 < w1 && w0 >= at && w0 < upto))
            for (int64_t s = s0; s < s1; ++s) {
                const int64_t u = head_units(seq_span(a, s), ROWS, p.group, UNIT);
                if (blockIdx.x == 0) p.first[s] = at;
                if (w0 < w1 && w0 >= at && w0 < at + u * a.n_kv_heads) { place[0] = s; place[1] = (w0 - at) / u; place[2] = (w0 - at) % u; }
                at += u * a.n_kv_heads;
            }
        if (blockIdx.x == 0 && tid == 0) p.first[a.n_seqs] = total;
        if (w0 == w1) return;
        __syncthreads();
        use.seq = place[0];
        use.head = (int)place[1];
        int64_t in = place[2];
        use.v = seq_span(a, use.seq);
        use.tiles = tiles_of(use.v, ROWS, p.group);
        use.tile = 0;
        load_segment<ROWS, UNIT>(p, use);
        while (in >= use.units) { in -= use.units; ++use.tile; load_segment<ROWS, UNIT>(p, use); }
        use.unit = (int)in;
    }
    const int64_t count = w1 - w0;

    // ---- loads: a stage of this key group is 16 keys, whose rows lane l & 15 finds ----
    const uint32_t ring = smem_u32(smem) + kg * S * STAGE;
    Cursor get = use;
    int64_t got = 0;
    int page = 0, pos = 0;          // of key l & 15 of the stage after the one being asked for
    bool page_ok = false, key_ok = false;
    auto look = [&]() {             // the page of the stage at `get`
        const int key = (get.unit * KG + kg) * 16 + (lane & 15);
        key_ok = got < count && key < get.keys;
        pos = key / a.page_size;
        page_ok = key_ok && pos < a.table_width;
        page = page_ok ? a.page_table[get.seq * a.ld_table + pos] : 0;
        pos = key - pos * a.page_size;
    };
    auto ask = [&](int slot) {      // copies the stage that look() has seen, then looks at the next
        if (got < count) {
            const bool ok = page_ok && page >= 0 && page < a.n_pages;
            const uint32_t bad = __ballot_sync(~0u, key_ok && !ok) & 0xffffu;
            const int64_t koff = ok ? page * a.k_strides[0] + pos * a.k_strides[1] : 0, voff = ok ? page * a.v_strides[0] + pos * a.v_strides[1] : 0;
            const uint32_t real = __ballot_sync(~0u, ok) & 0xffffu;
            const __nv_bfloat16 *k = (const __nv_bfloat16 *)a.k_pages + get.head * a.k_strides[2], *v = (const __nv_bfloat16 *)a.v_pages + get.head * a.v_strides[2];
            const uint32_t dst = ring + slot * STAGE;
#pragma unroll
            for (int i = 0; i < 16 * CH / 32 / RG; ++i) {
                const int piece = (i * RG + rg) * 32 + lane, row = piece / CH, c = piece % CH;
                const uint32_t to = dst + row * (D * 2) + (((c & ~7) | ((c ^ row) & 7)) << 4);
                const int64_t ko = __shfl_sync(~0u, koff, row), vo = __shfl_sync(~0u, voff, row);
                cp_async16(to, k + ko + c * 8, real >> row & 1);
                cp_async16(to + 16 * D * 2, v + vo + c * 8, real >> row & 1);
            }
            if (rg == 0 && lane == 0) {
                bad_sm[kg * S + slot] = bad;
                if (bad) atomicMax(p.status, GQ_DEV_BAD_SHAPE);
            }
            ++got;
            if (++get.unit == get.units && got < count) next_segment<ROWS, UNIT>(p, get);
            look();
        }
        cp_async_commit();
    };
    look();
    for (int i = 0; i < S - 1; ++i) ask(i);

    float o[NT][4], top[2], sum[2];
    uint32_t qf[QREG ? KK : 1][4];
    int lim[2], lim_first = 0;     // keys that this lane's rows see, and the tile's first row
    bool fresh = true;
    int unit0 = 0;                 // this block's first unit of the segment
    int slot = 0;
    const uint32_t q_addr = smem_u32(q_sm) + rg * 16 * D * 2;

    for (int64_t it = 0; it < count; ++it) {
        if (fresh) {
            fresh = false;
            unit0 = use.unit;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
            const int64_t rows = (int64_t)use.v.n * p.group, row0 = (int64_t)use.tile * ROWS + rg * 16;
            const __nv_bfloat16 *src[2];
            bool have[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[j] = -INFINITY;
                sum[j] = 0.0f;
                const int64_t r = row0 + g + 8 * j;
                have[j] = r < rows;
                const int i = have[j] ? (int)(r / p.group) : 0, h = have[j] ? (int)(r % p.group) : 0;
                lim[j] = use.v.len - use.v.n + i + 1;
                src[j] = (const __nv_bfloat16 *)a.q + (use.v.tok0 + i) * a.q_strides[0] + (use.head * p.group + h) * a.q_strides[1];
            }
            lim_first = use.v.len - use.v.n + (int)(((int64_t)use.tile * ROWS) / p.group) + 1;
            if constexpr (QREG) {
#pragma unroll
                for (int i = 0; i < KK; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) qf[i][j] = have[j & 1] ? *(const uint32_t *)(src[j & 1] + i * 16 + (j >> 1) * 8 + t * 2) : 0u;
            } else {
                // the rows of this row group, once for its KG warps: before the barrier of this iteration, behind that of the last merge
                for (int i = kg * 32 + lane; i < 16 * CH; i += 32 * KG) {
                    const int row = i / CH, c = i % CH;
                    const int64_t r = row0 + row;
                    uint4 val = make_uint4(0, 0, 0, 0);
                    if (r < rows)
                        val = *(const uint4 *)((const __nv_bfloat16 *)a.q + (use.v.tok0 + r / p.group) * a.q_strides[0] + (use.head * p.group + r % p.group) * a.q_strides[1] + c * 8);
                    *(uint4 *)(q_sm + (rg * 16 + row) * (D * 2) + (((c & ~7) | ((c ^ row) & 7)) << 4)) = val;
                }
                __syncthreads();
            }
        }
        cp_async_wait<S - 2>();
        if constexpr (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * RG) : "memory");
        else __syncwarp();
        ask((slot + S - 1) % S);

        // ---- scores of 16 keys ----
        const uint32_t ks = ring + slot * STAGE, vs = ks + 16 * D * 2;
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        {
            const int row = (lane >> 4) * 8 + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
            for (int i = 0; i < KK; ++i) {
                const int c = 2 * i + half;
                uint32_t kf[4];
                ldsm4(kf, ks + row * (D * 2) + (((c & ~7) | ((c ^ row) & 7)) << 4));
                if constexpr (QREG) {
                    mma_bf16(s[0], qf[i], kf[0], kf[1]);
                    mma_bf16(s[1], qf[i], kf[2], kf[3]);
                } else {
                    const int qr = ((lane >> 3) & 1) * 8 + (lane & 7), qc = 2 * i + (lane >> 4);
                    uint32_t q4[4];
                    ldsm4(q4, q_addr + qr * (D * 2) + (((qc & ~7) | ((qc ^ qr) & 7)) << 4));
                    mma_bf16(s[0], q4, kf[0], kf[1]);
                    mma_bf16(s[1], q4, kf[2], kf[3]);
                }
            }
        }
        const int key0 = (use.unit * KG + kg) * 16;
        const uint32_t bad = bad_sm[kg * S + slot];
        const bool edge = key0 + 16 > lim_first || bad;        // a row of the tile does not see all of these keys, or a page is missing
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] *= p.scale2;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = i * 8 + t * 2 + (j & 1);
                    if (bad >> at & 1) s[i][j] = __int_as_float(0x7fc00000);
                    if (key0 + at >= lim[j >> 1]) s[i][j] = -INFINITY;
                }
        }
        // ---- running maximum and sum ----
        float next[2], ref[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float m = fmaxf(fmaxf(s[0][2 * j], s[0][2 * j + 1]), fmaxf(s[1][2 * j], s[1][2 * j + 1]));
            m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
            m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
            next[j] = fmaxf(top[j], m);
            ref[j] = next[j] == -INFINITY ? 0.0f : next[j];
        }
        if (__any_sync(~0u, next[0] > top[0] || next[1] > top[1])) {
            const float keep[2] = {ex2(top[0] - ref[0]), ex2(top[1] - ref[1])};
#pragma unroll
            for (int j = 0; j < 2; ++j) { top[j] = next[j]; sum[j] *= keep[j]; }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] *= keep[j >> 1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[i][j] = ex2(s[i][j] - ref[j >> 1]); sum[j >> 1] += s[i][j]; }
        // ---- p v ----
        uint32_t big[4], small[4], vm0 = ~0u, vm1 = ~0u;
        // Keys that some rows of the tile see and others do not: a masked probability of 0 would still make NaN of an infinite value, so these keys stay out of the MMA and are
        // added row by row.  There are fewer of them in all than new tokens in the tile.
        const bool split = edge && lim_first < use.keys && key0 + 16 > lim_first;
        const int from = split ? max(lim_first - key0, 0) : 16, to = split ? min(use.keys - key0, 16) : 16;
        if (split) {
            const int at = t * 2;
            vm0 = (at < from ? 0xffffu : 0u) | (at + 1 < from ? 0xffff0000u : 0u);
            vm1 = (at + 8 < from ? 0xffffu : 0u) | (at + 9 < from ? 0xffff0000u : 0u);
            for (int x = from; x < to; ++x) {
                const int owner = (lane & ~3) | ((x & 7) >> 1), i = x >> 3;
                const float pa = __shfl_sync(~0u, i ? ((x & 1) ? s[1][1] : s[1][0]) : ((x & 1) ? s[0][1] : s[0][0]), owner);
                const float pb = __shfl_sync(~0u, i ? ((x & 1) ? s[1][3] : s[1][2]) : ((x & 1) ? s[0][3] : s[0][2]), owner);
                const bool see_a = key0 + x < lim[0], see_b = key0 + x < lim[1];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t w = *(const uint32_t *)(smem + (vs - smem_u32(smem)) + x * (D * 2) + (((n & ~7) | ((n ^ x) & 7)) << 4) + t * 4);
                    const float v0 = __uint_as_float(w << 16), v1 = __uint_as_float(w & 0xffff0000u);
                    if (see_a) { o[n][0] += pa * v0; o[n][1] += pa * v1; }
                    if (see_b) { o[n][2] += pb * v0; o[n][3] += pb * v1; }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i * 8 + t * 2 + (j & 1) >= from) s[i][j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) bf16_parts(s[j >> 1][2 * (j & 1)], s[j >> 1][2 * (j & 1) + 1], big[j], small[j]);
        {
            const int row = ((lane >> 3) & 1) * 8 + (lane & 7), half = lane >> 4;
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                const int c = n + half;
                uint32_t vf[4];
                ldsm4_t(vf, vs + row * (D * 2) + (((c & ~7) | ((c ^ row) & 7)) << 4));
                if (split) { vf[0] &= vm0; vf[1] &= vm1; vf[2] &= vm0; vf[3] &= vm1; }
                mma_bf16(o[n], big, vf[0], vf[1]);
                mma_bf16(o[n + 1], big, vf[2], vf[3]);
                mma_bf16(o[n], small, vf[0], vf[1]);
                mma_bf16(o[n + 1], small, vf[2], vf[3]);
            }
        }
        slot = (slot + 1) % S;
        ++use.unit;
        if (use.unit != use.units && it + 1 != count) continue;

        // ---- the end of this block's part of a segment: key groups joined, from the last to the first ----
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            sum[j] += __shfl_xor_sync(~0u, sum[j], 1);
            sum[j] += __shfl_xor_sync(~0u, sum[j], 2);
        }
        if constexpr (KG > 1) {
            if (t == 0)
                for (int j = 0; j < 2; ++j) stat_sm[kg * ROWS + rg * 16 + g + 8 * j] = make_float2(top[j], sum[j]);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float m = -INFINITY, l = 0.0f;
                for (int x = 0; x < KG; ++x) m = fmaxf(m, stat_sm[x * ROWS + rg * 16 + g + 8 * j].x);
                const float r = m == -INFINITY ? 0.0f : m;
                for (int x = 0; x < KG; ++x) {
                    const float2 st = stat_sm[x * ROWS + rg * 16 + g + 8 * j];
                    l += st.y * ex2(st.x - r);
                }
                const float keep = ex2(top[j] - r);
#pragma unroll
                for (int n = 0; n < NT; ++n) { o[n][2 * j] *= keep; o[n][2 * j + 1] *= keep; }
                top[j] = m;
                sum[j] = l;
            }
            float4 *box = (float4 *)merge + rg * 16 * D / 4 + lane;
            for (int x = KG - 1; x > 0; --x) {
                if (kg == x)
#pragma unroll
                    for (int n = 0; n < NT; ++n) box[n * 32] = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
                __syncthreads();
                if (kg == x - 1)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float4 v = box[n * 32];
                        o[n][0] += v.x; o[n][1] += v.y; o[n][2] += v.z; o[n][3] += v.w;
                    }
                __syncthreads();
            }
        }
        if (kg == 0) {
            const bool whole = unit0 == 0 && use.unit == use.units;
            const int64_t part = 2 * (int64_t)blockIdx.x + (unit0 == 0), rows = (int64_t)use.v.n * p.group;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t r = (int64_t)use.tile * ROWS + rg * 16 + g + 8 * j;
                if (r >= rows) continue;
                if (whole) {
                    const int64_t tok = use.v.tok0 + r / p.group, h = use.head * p.group + r % p.group;
                    __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + tok * a.out_strides[0] + h * a.out_strides[1] + t * 2;
                    const __nv_bfloat16 *gate = a.gate ? (const __nv_bfloat16 *)a.gate + tok * a.gate_strides[0] + h * a.gate_strides[1] + t * 2 : nullptr;
                    const float inv = sum[j] == 0.0f ? 0.0f : 1.0f / sum[j];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float v = o[n][2 * j + x] * inv;
                            if (gate) v /= 1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[n * 8 + x]));
                            dst[n * 8 + x] = __float2bfloat16_rn(v);
                        }
                } else {
                    const int64_t at = part * ROWS + rg * 16 + g + 8 * j;
                    if (t == 0) p.stats[at] = make_float2(top[j], sum[j]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) *(float2 *)(p.parts + at * D + n * 8 + t * 2) = make_float2(o[n][2 * j], o[n][2 * j + 1]);
                }
            }
        }
        fresh = true;
        if (it + 1 != count) next_segment<ROWS, UNIT>(p, use);
    }
    cp_async_wait<0>();
}

// The rows whose keys lie in several blocks' ranges, or that see none: one block of 128 threads to a token's query head, its threads in sets of head_dim / 4 that
// take the parts in turn.
template <int D>
__global__ void __launch_bounds__(128) join_parts_kernel(const __grid_constant__ PagedParams p, int rows_of_tile, int unit) {
    constexpr int LANES = D / 4, SETS = 128 / LANES;
    __shared__ float4 acc[SETS][LANES];
    __shared__ float red[4];
    const gq_attention_args &a = p.a;
    const int64_t tok = blockIdx.x;
    const int h = blockIdx.y, kvh = h / p.group, set = threadIdx.x / LANES, at4 = threadIdx.x % LANES;
    pdl_wait();
    int64_t s = 0;
    if (a.q_starts) {
        int64_t hi = a.n_seqs;                    // the last sequence that starts at or before the token
        while (s + 1 < hi) {
            const int64_t mid = (s + hi) / 2;
            if (a.q_starts[mid] <= tok) s = mid; else hi = mid;
        }
    } else s = tok / (a.T / a.n_seqs);
    const SeqSpan v = seq_span(a, s);
    if (tok < v.tok0 || tok >= v.tok0 + v.n) return;          // nobody's row
    const int64_t row = (tok - v.tok0) * p.group + h % p.group;
    const int tile = (int)(row / rows_of_tile);
    int64_t first = p.first[s] + (int64_t)kvh * head_units(v, rows_of_tile, p.group, unit);
    for (int i = 0; i < tile; ++i) first += (tile_keys(v, i, rows_of_tile, p.group) + unit - 1) / unit;
    const int64_t units = (tile_keys(v, tile, rows_of_tile, p.group) + unit - 1) / unit, total = p.first[a.n_seqs];
    const int64_t blocks = min((int64_t)p.blocks, max(total, (int64_t)1));
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    if (units > 0) {
        const int64_t c0 = ((first + 1) * blocks - 1) / total, c1 = min(((first + units) * blocks - 1) / total, blocks - 1);
        if (c0 == c1) return;                     // finished by its block
        const int64_t r = row % rows_of_tile;
        auto part = [&](int64_t c) { return (2 * c + (c == c0)) * rows_of_tile + r; };
        float top = -INFINITY;
        for (int64_t c = c0 + threadIdx.x; c <= c1; c += 128) top = fmaxf(top, p.stats[part(c)].x);
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
        for (int64_t c = c0 + set; c <= c1; c += SETS) {
            const int64_t q = part(c);
            const float2 st = p.stats[q];
            const float4 w = *(const float4 *)(p.parts + q * D + at4 * 4);
            const float f = ex2(st.x - ref);
            sum += f * st.y;
            o.x += f * w.x; o.y += f * w.y; o.z += f * w.z; o.w += f * w.w;
        }
        __shared__ float sums[SETS];
        acc[set][at4] = o;
        if (at4 == 0) sums[set] = sum;
        __syncthreads();
        if (set) return;
        for (int x = 1; x < SETS; ++x) {
            const float4 w = acc[x][at4];
            o.x += w.x; o.y += w.y; o.z += w.z; o.w += w.w;
            sum += sums[x];
        }
    }
    if (set) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float val[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + tok * a.out_strides[0] + h * a.out_strides[1] + at4 * 4;
    const __nv_bfloat16 *gate = a.gate ? (const __nv_bfloat16 *)a.gate + tok * a.gate_strides[0] + h * a.gate_strides[1] + at4 * 4 : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = __float2bfloat16_rn(gate ? val[i] / (1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[i]))) : val[i]);
}

}  // namespace gq
