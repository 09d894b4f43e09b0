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
#include "gq_bf16.cuh"

namespace gq {

struct PagedParams {
    gq_attention_args a;
    int *status;
    float2 *stats;          // workspace: [2 G][rows of a tile]: maximum, sum
    float *parts;           // [2 G][rows of a tile][head_dim]
    int group, blocks, max_keys;        // query heads of a kv head; blocks the GPU holds; keys that the page table has room for
    int per_seq;            // tokens of a sequence where all have the same
    int whole;              // pages hold whole stages of 16 keys
    uint32_t page_mul, page_shift;      // key / page_size = key * page_mul >> page_shift, for keys below 2^31
    float scale2;           // scale * log2 e
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two probabilities as bf16 and what that rounding left, as bf16
__device__ __forceinline__ void bf16_parts(float lo, float hi, uint32_t &big, uint32_t &small) {
    big = bf16_pair(lo, hi);
    small = bf16_pair(lo - __uint_as_float(big << 16), hi - __uint_as_float(big & 0xffff0000u));
}

// an 8 x 8 tile of 16-bit values, a row to four lanes, turned over
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// A sequence's tokens and keys, and how its rows and keys are cut
struct SeqSpan {
    int64_t tok0;     // its first token
    int n, len;       // new tokens, keys
};
__device__ __forceinline__ SeqSpan seq_span(const PagedParams &p, int64_t s) {
    const gq_attention_args &a = p.a;
    SeqSpan v;
    if (a.q_starts) {
        const int64_t q0 = min(max((int64_t)a.q_starts[s], (int64_t)0), a.T), q1 = min(max((int64_t)a.q_starts[s + 1], q0), a.T);
        v.tok0 = q0; v.n = (int)(q1 - q0);
    } else {
        v.n = p.per_seq; v.tok0 = s * v.n;
    }
    v.len = min(max(a.lens[s], 0), p.max_keys + v.n);      // with more keys than the table has, every token sees a missing one
    return v;
}
// keys that a tile's last row sees (a sequence's rows, its tokens times the group, are fewer than 2^30)
__device__ __forceinline__ int tile_keys(const SeqSpan &v, int tile, int rows, int group) {
    const int last = min(v.n, (int)(((unsigned)(tile + 1) * rows - 1) / (unsigned)group) + 1);       // tokens up to the tile's last
    return max(0, v.len - v.n + last);
}
__device__ __forceinline__ int tiles_of(const SeqSpan &v, int rows, int group) { return (int)(((unsigned)v.n * group + rows - 1) / rows); }
__device__ __forceinline__ int64_t head_units(const SeqSpan &v, int rows, int group, int unit) {
    if (v.n * group <= rows) return v.n ? (unsigned)(v.len + unit - 1) / unit : 0;
    int64_t u = 0;
    for (int t = 0, n = tiles_of(v, rows, group); t < n; ++t) u += (unsigned)(tile_keys(v, t, rows, group) + unit - 1) / unit;
    return u;
}
// n / d, in 32 bits where both fit: the 64-bit division is a hundred instructions
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
    return ((uint64_t)n | (uint64_t)d) >> 32 ? (int64_t)((uint64_t)n / (uint64_t)d) : (int64_t)((uint32_t)n / (uint32_t)d);
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
                    c.v = seq_span(p, c.seq);
                    c.tiles = tiles_of(c.v, ROWS, p.group);
                } while (c.tiles == 0);
            }
        }
        load_segment<ROWS, UNIT>(p, c);
    } while (c.units == 0);
}

// The line of all units as one warp sees it: lane l counts the sequences [l each, (l + 1) each)
struct Line {
    int64_t mine, upto, total;      // units of this lane's sequences, of those and all before, of all
    int64_t s0, s1;
};
template <int ROWS, int UNIT> __device__ __forceinline__ Line count_units(const PagedParams &p, int lane) {
    Line l;
    const int64_t each = (p.a.n_seqs + 31) / 32;
    l.s0 = min(lane * each, p.a.n_seqs);
    l.s1 = min(l.s0 + each, p.a.n_seqs);
    l.mine = 0;
    for (int64_t s = l.s0; s < l.s1; ++s) l.mine += head_units(seq_span(p, s), ROWS, p.group, UNIT) * p.a.n_kv_heads;
    l.upto = l.mine;
    for (int o = 1; o < 32; o *= 2) {
        const int64_t v = __shfl_up_sync(~0u, l.upto, o);
        if (lane >= o) l.upto += v;
    }
    l.total = __shfl_sync(~0u, l.upto, 31);
    return l;
}
// How the line is cut: block c's units are [start(c), start(c + 1)), the first `more` blocks have one more than the others
struct Cut {
    int64_t each, more, blocks;
    __device__ __forceinline__ int64_t start(int64_t c) const { return min(c, blocks) * each + min(c, more); }
    __device__ __forceinline__ int64_t block_of(int64_t x) const {
        const int64_t large = more * (each + 1);
        return x < large ? quotient(x, each + 1) : more + quotient(x - large, max(each, (int64_t)1));
    }
};
__device__ __forceinline__ Cut cut_line(const PagedParams &p, int64_t total) {
    Cut c;
    c.blocks = p.blocks;
    c.each = quotient(total, c.blocks);
    c.more = total - c.each * c.blocks;
    return c;
}
// the segment of unit x of the line (0 <= x < total)
template <int ROWS, int UNIT> __device__ __forceinline__ void locate(const PagedParams &p, const Line &l, int64_t x, int lane, Cursor &c) {
    const int owner = __ffs(__ballot_sync(~0u, x < l.upto)) - 1;
    int64_t seq = 0, in = 0;
    if (lane == owner) {
        in = x - (l.upto - l.mine);
        for (seq = l.s0;; ++seq) {
            const int64_t u = head_units(seq_span(p, seq), ROWS, p.group, UNIT) * p.a.n_kv_heads;
            if (in < u) break;
            in -= u;
        }
    }
    c.seq = __shfl_sync(~0u, seq, owner);
    in = __shfl_sync(~0u, in, owner);
    c.v = seq_span(p, c.seq);
    c.tiles = tiles_of(c.v, ROWS, p.group);
    const int64_t per_head = head_units(c.v, ROWS, p.group, UNIT);
    c.head = (int)quotient(in, per_head);
    in -= c.head * per_head;
    c.tile = 0;
    load_segment<ROWS, UNIT>(p, c);
    while (in >= c.units) { in -= c.units; ++c.tile; load_segment<ROWS, UNIT>(p, c); }
    c.unit = (int)in;
}

template <int D, int RG, int KG, int S> struct PagedShape {
    static constexpr int THREADS = 32 * RG * KG, ROWS = 8 * RG, UNIT = 16 * KG;
    static constexpr int PITCH = D * 2 + 16;                                    // bytes of a row in shared memory: eight rows' chunks in different banks
    static constexpr int STAGE = 2 * 16 * PITCH;                                // keys and values of 16 keys
    static constexpr int TURNS = RG > 2 ? 2 : 1;                                // a key group's output goes through the stage it used last, in as many turns
    static constexpr int RING = KG * S * STAGE, STATS = KG > 1 ? KG * ROWS * 8 : 0;
    static_assert(ROWS * D * 4 / TURNS <= STAGE && (D / 16) % (KG * TURNS) == 0, "the key groups share the dimensions of an output out");
    static constexpr int SMEM = RING + STATS + RG * KG * 256;
};

template <int D, int RG, int KG, int S>
__global__ void __launch_bounds__(32 * RG * KG) paged_attention_kernel(const __grid_constant__ PagedParams p) {
    using Shape = PagedShape<D, RG, KG, S>;
    constexpr int ROWS = Shape::ROWS, UNIT = Shape::UNIT, STAGE = Shape::STAGE, PITCH = Shape::PITCH, CH = D / 8, MT = D / 16, WARPS = RG * KG;
    extern __shared__ __align__(128) uint8_t smem[];
    float2 *stat_sm = (float2 *)(smem + Shape::RING);
    longlong2 *row_sm = (longlong2 *)((uint8_t *)stat_sm + Shape::STATS);       // [warp][16]: bytes to the keys and values of the stage being asked for
    const gq_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, rg = warp % RG, kg = warp / RG, g = lane / 4, t = lane % 4;
    pdl_wait();
    pdl_trigger();

    // ---- this block's units (every warp counts for itself) ----
    Cursor use;
    int64_t w0, w1;
    {
        const Line line = count_units<ROWS, UNIT>(p, lane);
        const Cut cut = cut_line(p, line.total);
        w0 = cut.start(blockIdx.x);
        w1 = cut.start(blockIdx.x + 1);
        if (w0 < w1) locate<ROWS, UNIT>(p, line, w0, lane, use);
    }
    // tokens that see no key: their tiles have no units, and belong to the last blocks, which are idle first
    auto zeros = [&]() {
        for (int64_t s = gridDim.x - 1 - blockIdx.x; s < a.n_seqs; s += gridDim.x) {
            const SeqSpan v = seq_span(p, s);
            for (int tile = 0, n = tiles_of(v, ROWS, p.group); tile < n && tile_keys(v, tile, ROWS, p.group) == 0; ++tile)
                for (int r = tile * ROWS, end = min(r + ROWS, v.n * p.group); r < end; ++r)
                    for (int i = tid; i < a.n_kv_heads * D; i += Shape::THREADS)
                        ((__nv_bfloat16 *)a.out)[(v.tok0 + r / p.group) * a.out_strides[0] + ((i / D) * p.group + r % p.group) * a.out_strides[1] + i % D] = __float2bfloat16_rn(0.0f);
        }
    };
    if (w0 == w1) { zeros(); return; }
    const int count = (int)(w1 - w0);

    // ---- loads: a stage of this key group is 16 keys ----
    const uint32_t ring = smem_u32(smem) + kg * S * STAGE;
    constexpr int PER = 32 / CH, COPIES = 16 * CH / 32;        // rows that 32 lanes copy at once, 16 bytes each; turns for a stage
    const int copy_row = lane / CH, copy_c = lane % CH;
    const uint32_t copy_to = ring + copy_row * PITCH + copy_c * 16;
    Cursor get = use;
    int got = 0, page = 0, pos = 0;        // of the next stage to ask for: the page and row of its first key, or (pages that end inside a stage) of key lane & 15
    bool page_ok = false, key_ok = false;
    uint32_t k_step = (uint32_t)a.k_strides[1] * 2, v_step = (uint32_t)a.v_strides[1] * 2;      // bytes between rows of a page (whole pages: below 2^32)
    const char *k_head, *v_head;
    auto heads = [&]() {
        k_head = (const char *)((const __nv_bfloat16 *)a.k_pages + get.head * a.k_strides[2] + copy_c * 8 + (p.whole ? copy_row * a.k_strides[1] : 0));
        v_head = (const char *)((const __nv_bfloat16 *)a.v_pages + get.head * a.v_strides[2] + copy_c * 8 + (p.whole ? copy_row * a.v_strides[1] : 0));
    };
    auto look = [&]() {
        const int key = (get.unit * KG + kg) * 16 + (p.whole ? 0 : lane & 15);
        key_ok = got < count && key < get.keys;
        const int at = (int)((uint64_t)(uint32_t)key * p.page_mul >> p.page_shift);
        page_ok = key_ok && at < a.table_width;
        page = page_ok ? a.page_table[get.seq * a.ld_table + at] : 0;
        pos = key - at * a.page_size;
    };
    longlong2 *rows_at = row_sm + warp * 16;
    uint64_t missing = 0;           // of the stages asked for and not used yet, 16 bits each, the next one lowest: keys whose page is missing
    auto ask = [&](int slot) {      // copies the stage that look() has seen, then looks at the next
        uint32_t bad = 0;
        if (got < count) {
            const bool ok = page_ok && page >= 0 && page < a.n_pages;
            const uint32_t dst = copy_to + slot * STAGE;
            if (p.whole) {          // the stage lies in one page
                const int seen = min(get.keys - (get.unit * KG + kg) * 16, 16), real = ok ? seen : 0;
                const char *k = k_head + (page * a.k_strides[0] + pos * a.k_strides[1]) * 2, *v = v_head + (page * a.v_strides[0] + pos * a.v_strides[1]) * 2;
                if (real == 16) {
#pragma unroll
                    for (int i = 0; i < (COPIES + RG - 1) / RG; ++i) {
                        if (COPIES % RG && i * RG + rg >= COPIES) break;
                        const uint32_t row = (RG > 1 ? i * RG + rg : i) * PER;
                        cp_async16(dst + row * PITCH, k + (uint64_t)row * k_step);
                        cp_async16(dst + (16 + row) * PITCH, v + (uint64_t)row * v_step);
                    }
                } else {
                    bad = ok || seen <= 0 ? 0u : (1u << seen) - 1;
#pragma unroll 1
                    for (int i = rg; i < COPIES; i += RG) {
                        const uint32_t row = i * PER;
                        const bool is = (int)row + copy_row < real;
                        cp_async16(dst + row * PITCH, is ? k + (uint64_t)row * k_step : (const char *)a.k_pages, is);
                        cp_async16(dst + (16 + row) * PITCH, is ? v + (uint64_t)row * v_step : (const char *)a.v_pages, is);
                    }
                }
            } else {                // lane l finds key l & 15
                bad = __ballot_sync(~0u, key_ok && !ok) & 0xffffu;
                const uint32_t real = __ballot_sync(~0u, ok);
                __syncwarp();
                if (lane < 16) rows_at[lane] = ok ? make_longlong2(2 * (page * a.k_strides[0] + pos * a.k_strides[1]), 2 * (page * a.v_strides[0] + pos * a.v_strides[1])) : make_longlong2(0, 0);
                __syncwarp();
#pragma unroll 2
                for (int i = rg; i < COPIES; i += RG) {
                    const int row = i * PER;
                    const longlong2 at = rows_at[row + copy_row];
                    const bool is = real >> (row + copy_row) & 1;
                    cp_async16(dst + row * PITCH, k_head + at.x, is);
                    cp_async16(dst + (16 + row) * PITCH, v_head + at.y, is);
                }
            }
            if (bad && lane == 0) atomicMax(p.status, GQ_DEV_BAD_SHAPE);
            ++got;
            if (++get.unit == get.units && got < count) { next_segment<ROWS, UNIT>(p, get); heads(); }
            look();
        }
        missing = missing >> 16 | (uint64_t)bad << (16 * (S - 2));
        cp_async_commit();
    };
    heads();
    look();
#pragma unroll 1
    for (int i = 0; i < S - 1; ++i) ask(i);
    zeros();

    // Transposed products: keys (or dimensions) on M, the eight query rows of the warp on N.  A lane holds, of a score tile, keys g and g + 8 of queries 2 t and 2 t + 1; of the
    // output, dimensions 16 i + g and 16 i + g + 8 of the same two queries.
    float o[MT][4], top[2], sum[2];
    uint32_t qf[MT][2];
    int lim[2], lim_first = 0;     // keys that this lane's queries see, and the tile's first row
    int slot = 0;
    // where this lane's row of an ldmatrix starts: keys (rows 0-7, 8-15 of one chunk, then of the next), values (transposed: two chunks of rows 0-7, then of 8-15)
    const uint32_t k_lane = (((lane >> 3) & 1) * 8 + (lane & 7)) * PITCH + (lane >> 4) * 16, v_lane = (16 + (lane >> 4) * 8 + (lane & 7)) * PITCH + ((lane >> 3) & 1) * 16;

    for (int it = 0;;) {
        const int unit0 = use.unit;         // this block's first unit of the segment
        {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
            const int rows = use.v.n * p.group, row0 = use.tile * ROWS + rg * 8;
            const int before = use.v.len - use.v.n + 1;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[j] = -INFINITY;
                sum[j] = 0.0f;
                lim[j] = before + (unsigned)min(row0 + 2 * t + j, rows - 1) / (unsigned)p.group;
            }
            lim_first = before + (unsigned)(use.tile * ROWS) / (unsigned)p.group;
            const int r = row0 + g, i = (unsigned)r / (unsigned)p.group;
            const uint32_t *src = (const uint32_t *)((const __nv_bfloat16 *)a.q + (use.v.tok0 + i) * a.q_strides[0] + (use.head * p.group + (r - i * p.group)) * a.q_strides[1]) + t;
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int j = 0; j < 2; ++j) qf[x][j] = r < rows ? src[x * 8 + j * 4] : 0u;
        }
        for (const int end = min(use.units, use.unit + count - it); use.unit < end; ++use.unit) {
            cp_async_wait<S - 2>();
            if constexpr (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * RG) : "memory");
            else __syncwarp();
            const uint32_t bad = (uint32_t)missing & 0xffffu;
            ask(slot == 0 ? S - 1 : slot - 1);

            // ---- scores of 16 keys ----
            const uint32_t stage = ring + slot * STAGE;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t kf[4];
                ldsm4(kf, stage + k_lane + i * 32);
                mma_bf16(i & 1 ? s2 : s, kf, qf[i][0], qf[i][1]);
            }
            const int key0 = (use.unit * KG + kg) * 16;
            const bool edge = key0 + 16 > lim_first || bad;        // a row of the tile does not see all of these keys, or a page is missing
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = (s[j] + s2[j]) * p.scale2;
            if (edge) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = g + (j >> 1) * 8;
                    if (bad >> at & 1) s[j] = __int_as_float(0x7fc00000);
                    if (key0 + at >= lim[j & 1]) s[j] = -INFINITY;
                }
            }
            // ---- running maximum and sum ----
            float next[2], ref[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float m = fmaxf(s[j], s[j + 2]);
                m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                next[j] = fmaxf(top[j], m);
                ref[j] = next[j] == -INFINITY ? 0.0f : next[j];
            }
            if (__any_sync(~0u, next[0] > top[0] || next[1] > top[1])) {
                const float keep[2] = {ex2(top[0] - ref[0]), ex2(top[1] - ref[1])};
#pragma unroll
                for (int j = 0; j < 2; ++j) { top[j] = next[j]; sum[j] *= keep[j]; }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[i][j] *= keep[j & 1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { s[j] = ex2(s[j] - ref[j & 1]); sum[j & 1] += s[j]; }
            // ---- p v ----
            // Keys that some rows of the tile see and others do not: a masked probability of 0 would still make NaN of an infinite value, so these keys stay out of the MMA and are
            // added row by row.  There are fewer of them in all than new tokens in the tile.
            const bool split = edge && lim_first < use.keys;
            const int from = split ? max(lim_first - key0, 0) : 16;
            if (split) {
                const int to = min(use.keys - key0, 16);
                for (int x = from; x < to; ++x) {
                    const int owner = (x & 7) * 4 + t;
                    const float pa = __shfl_sync(~0u, x & 8 ? s[2] : s[0], owner), pb = __shfl_sync(~0u, x & 8 ? s[3] : s[1], owner);
                    const bool see_a = key0 + x < lim[0], see_b = key0 + x < lim[1];
                    const __nv_bfloat16 *v = (const __nv_bfloat16 *)(smem + (stage - smem_u32(smem)) + (16 + x) * PITCH) + g;
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float val = __bfloat162float(v[i * 16 + j * 8]);
                            if (see_a) o[i][2 * j] += pa * val;
                            if (see_b) o[i][2 * j + 1] += pb * val;
                        }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (g + (j >> 1) * 8 >= from) s[j] = 0.0f;
            }
            // the probabilities of eight keys, turned over: queries on g, keys 2 t and 2 t + 1, as the B operand has them
            uint32_t big[2], small[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16_parts(s[2 * j], s[2 * j + 1], big[j], small[j]);
                big[j] = transpose8(big[j]);
                small[j] = transpose8(small[j]);
            }
            if (split) {
                const uint32_t vm0 = (2 * t < from ? 0xffffu : 0u) | (2 * t + 1 < from ? 0xffff0000u : 0u), vm1 = (2 * t + 8 < from ? 0xffffu : 0u) | (2 * t + 9 < from ? 0xffff0000u : 0u);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    uint32_t vf[4];
                    ldsm4_t(vf, stage + v_lane + i * 32);
                    vf[0] &= vm0; vf[1] &= vm0; vf[2] &= vm1; vf[3] &= vm1;
                    mma_bf16(o[i], vf, big[0], big[1]);
                    mma_bf16(o[i], vf, small[0], small[1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    uint32_t vf[4];
                    ldsm4_t(vf, stage + v_lane + i * 32);
                    mma_bf16(o[i], vf, big[0], big[1]);
                    mma_bf16(o[i], vf, small[0], small[1]);
                }
            }
            if (++slot == S) slot = 0;
            ++it;
        }

        // ---- the end of this block's part of a segment: key groups joined, from the last to the first ----
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 4; x < 32; x *= 2) sum[j] += __shfl_xor_sync(~0u, sum[j], x);
        constexpr int MINE = MT / KG, TURNS = Shape::TURNS;       // dimension tiles that a key group adds up, the turns of the exchange
        float sum_o[MINE][4];
        if constexpr (KG > 1) {
            if (g == 0)
                for (int j = 0; j < 2; ++j) stat_sm[kg * ROWS + rg * 8 + 2 * t + j] = make_float2(top[j], sum[j]);
            const int used = (slot == 0 ? S - 1 : slot - 1) * STAGE;
            if constexpr (RG > 1) asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * RG) : "memory");      // nobody reads that stage any more
            else __syncwarp();
            float keep[KG][2];
#pragma unroll
            for (int h = 0; h < TURNS; ++h) {
                float4 *box = (float4 *)(smem + kg * S * STAGE + used) + rg * 2 * D / TURNS + lane;
#pragma unroll
                for (int i = 0; i < MT / TURNS; ++i) {
                    const float(&v)[4] = o[h * (MT / TURNS) + i];
                    box[i * 32] = make_float4(v[0], v[1], v[2], v[3]);
                }
                __syncthreads();
                if (h == 0) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 *st = stat_sm + rg * 8 + 2 * t + j;
                        float m = -INFINITY;
                        for (int x = 0; x < KG; ++x) m = fmaxf(m, st[x * ROWS].x);
                        const float r = m == -INFINITY ? 0.0f : m;
                        top[j] = m;
                        sum[j] = 0.0f;
#pragma unroll
                        for (int x = 0; x < KG; ++x) {
                            keep[x][j] = ex2(st[x * ROWS].x - r);
                            sum[j] += st[x * ROWS].y * keep[x][j];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MINE / TURNS; ++i) {
                    float(&v)[4] = sum_o[h * (MINE / TURNS) + i];
                    v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
                    for (int x = 0; x < KG; ++x) {
                        const float4 w = ((const float4 *)(smem + x * S * STAGE + used))[rg * 2 * D / TURNS + (i * KG + kg) * 32 + lane];
                        v[0] += w.x * keep[x][0]; v[1] += w.y * keep[x][1]; v[2] += w.z * keep[x][0]; v[3] += w.w * keep[x][1];
                    }
                }
                __syncthreads();            // the next turn, or the next stage, comes to the same place
            }
        } else {
#pragma unroll
            for (int i = 0; i < MINE; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum_o[i][j] = o[i][j];
        }
        auto dim_of = [&](int i) { return ((i / (MINE / TURNS)) * (MT / TURNS) + (i % (MINE / TURNS)) * KG + kg) * 16 + g; };       // of sum_o[i][0], [1]; 8 more: of [2], [3]
        {
            const bool whole = unit0 == 0 && use.unit == use.units;
            const int64_t part = 2 * (int64_t)blockIdx.x + (unit0 == 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = use.tile * ROWS + rg * 8 + 2 * t + j;
                if (r >= use.v.n * p.group) continue;
                if (whole) {
                    const int i0 = (unsigned)r / (unsigned)p.group;
                    const int64_t tok = use.v.tok0 + i0, h = use.head * p.group + (r - i0 * p.group);
                    __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + tok * a.out_strides[0] + h * a.out_strides[1];
                    const __nv_bfloat16 *gate = a.gate ? (const __nv_bfloat16 *)a.gate + tok * a.gate_strides[0] + h * a.gate_strides[1] : nullptr;
                    const float inv = sum[j] == 0.0f ? 0.0f : 1.0f / sum[j];
#pragma unroll
                    for (int i = 0; i < MINE; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int d = dim_of(i) + 8 * x;
                            float v = sum_o[i][2 * x + j] * inv;
                            if (gate) v /= 1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[d]));
                            dst[d] = __float2bfloat16_rn(v);
                        }
                } else {
                    const int64_t at = part * ROWS + rg * 8 + 2 * t + j;
                    if (g == 0 && kg == 0) p.stats[at] = make_float2(top[j], sum[j]);
#pragma unroll
                    for (int i = 0; i < MINE; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) p.parts[at * D + dim_of(i) + 8 * x] = sum_o[i][2 * x + j];
                }
            }
        }
        if (it == count) break;
        next_segment<ROWS, UNIT>(p, use);
    }
    cp_async_wait<0>();
}

// The segments that several blocks worked on: block c joins the one that starts in block c's range and ends behind it, each row by as many warps as there are, four parts of
// a warp in flight.  All but the parts themselves is found before the wait for the blocks that write them.
constexpr int JOIN_WARPS = 16;
template <int D, int ROWS, int UNIT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_parts_kernel(const __grid_constant__ PagedParams p) {
    constexpr int V = D / 32;                                   // values to a lane
    __shared__ float box[JOIN_WARPS][D];
    __shared__ float2 box_stats[JOIN_WARPS];
    const gq_attention_args &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int64_t end;            // the block of the segment's last unit
    Cursor c;
    {
        const Line line = count_units<ROWS, UNIT>(p, lane);
        const Cut cut = cut_line(p, line.total);
        const int64_t w0 = cut.start(blockIdx.x), w1 = cut.start(blockIdx.x + 1);
        if (w0 == w1) return;
        locate<ROWS, UNIT>(p, line, w1 - 1, lane, c);
        const int64_t first = w1 - 1 - c.unit;
        if (first < w0 || first + c.units == w1) return;
        end = min(cut.block_of(first + c.units - 1), cut.blocks - 1);
    }
    const int rows = min(ROWS, c.v.n * p.group - c.tile * ROWS), sets = max(JOIN_WARPS / rows, 1), set = warp / min(rows, JOIN_WARPS);
    pdl_wait();
    for (int r0 = 0; r0 < rows; r0 += JOIN_WARPS) {
        const int r = r0 + (rows < JOIN_WARPS ? warp % rows : warp);
        const bool mine = r < rows && set < sets;
        float o[V], sum = 0.0f, top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.0f;
        if (mine)
            for (int64_t b = (int64_t)blockIdx.x + set; b <= end; b += 4 * sets) {
                float2 st[4];
                float v[4][V];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int64_t of = b + x * sets, at = (2 * of + (of == (int64_t)blockIdx.x)) * ROWS + r;
                    const bool is = of <= end;
                    st[x] = is ? __ldcg(p.stats + at) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[x][i] = is ? __ldcg(p.parts + at * D + i * 32 + lane) : 0.0f;
                }
                const float next = fmaxf(fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), top), ref = next == -INFINITY ? 0.0f : next, keep = ex2(top - ref);
                top = next;
                sum *= keep;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] *= keep;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float f = ex2(st[x].x - ref);
                    sum += f * st[x].y;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] += f * v[x][i];
                }
            }
        if (sets > 1) {
            if (set > 0 && mine) {
#pragma unroll
                for (int i = 0; i < V; ++i) box[warp][i * 32 + lane] = o[i];
                if (lane == 0) box_stats[warp] = make_float2(top, sum);
            }
            __syncthreads();
            if (set == 0 && mine)
                for (int x = 1; x < sets; ++x) {
                    const float2 st = box_stats[warp + rows * x];
                    const float next = fmaxf(st.x, top), ref = next == -INFINITY ? 0.0f : next, keep = ex2(top - ref), f = ex2(st.x - ref);
                    top = next;
                    sum = sum * keep + st.y * f;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = o[i] * keep + box[warp + rows * x][i * 32 + lane] * f;
                }
        }
        if (set == 0 && mine) {
            const int row = c.tile * ROWS + r, i0 = (unsigned)row / (unsigned)p.group;
            const int64_t tok = c.v.tok0 + i0, h = c.head * p.group + (row - i0 * p.group);
            __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + tok * a.out_strides[0] + h * a.out_strides[1] + lane;
            const __nv_bfloat16 *gate = a.gate ? (const __nv_bfloat16 *)a.gate + tok * a.gate_strides[0] + h * a.gate_strides[1] + lane : nullptr;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = o[i] * inv;
                if (gate) v /= 1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[i * 32]));
                dst[i * 32] = __float2bfloat16_rn(v);
            }
        }
    }
}

}  // namespace gq
