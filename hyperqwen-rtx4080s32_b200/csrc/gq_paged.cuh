// Attention of a sequence's newest tokens over its keys and values in the pages of a cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp2(c q . k_j - m),  c = scale log2 e,  m near the running maximum: one pass over keys and values.
//
// Bound by the bytes of the cache: a key-value head's key and value are 4 head_dim bytes, and the rows that share them (the query heads of the group, times the new tokens)
// are few.  So the work is cut evenly by keys, not by sequences: the units of all (sequence, kv head, tile of rows) in a line, a unit being KG * 16 keys, and block c of G takes
// units [c W / G, (c + 1) W / G).  A segment that lies in one block is finished there; of the others each block leaves its unnormalised rows, maxima and sums
// in the workspace, and join_parts_kernel adds them in block order.  Every block finds its place from lens alone, so the host need not know them, and the order of all sums
// follows from the lengths and the number of SMs.
//
// A block is KG key groups.  A key group streams 16 keys at a time through a ring of S stages of its own in shared memory (cp.async, 16 bytes a lane; rows at a pitch of 2 head_dim + 16 bytes, so that
// ldmatrix meets no bank twice) and multiplies them by all rows of the tile, 8 NQ of them: scores as k q^T and outputs as v^T p^T (mma.sync m16n8k16, keys and dimensions on M), since the rows are
// what there are few of.  A key is read from shared memory once.  Heads of 256 are split over DG = 2 warps, which exchange their halves of the scores.  p enters as two bf16 parts (p and what its
// rounding left): one part would add an error as large as the output's own rounding, and leaving the second out gained 3 % at 8 x 8,192 keys and nothing elsewhere.  With one token of a few heads the
// loads are the bound, whatever multiplies.  With several tokens or chunks of prompts they are not, and the same transposed products would suit tcgen05 (128 keys or dimensions on M, the rows on N, scores and
// outputs in tensor memory); that has not been built.
//
// Measured (graph of calls, heads 40 / 8 of 128, bf16): 64 sequences of up to 16,384 keys 231 us = 6.1 TB/s of cache, 0.93 of a copy's rate; 131,072 keys of one 97 us, 5.5 TB/s: the SMs do not get
// their bytes equally fast (80 us in the middle, 97 the slowest), and the join takes 5.  8 of up to 8,192 21 us, 517 keys of one 7.6, of which a launch, the way to the first key and a join are 6.
// Chunks of prompts: 2,048 tokens 750 us = 57 TFLOP/s, 512 behind 7,680 keys 745 us = 112 TFLOP/s, 8,192 tokens 7.3 ms: tiles of 32 rows read the keys again and again, and every block walks all
// tiles in front of its first.  16 x 4 tokens of 24 / 4 heads of 256 109 us = 3.2 TB/s: two warps to a scheduler, each with a chain of 72 products, an exchange and the probabilities of 24 rows for every 16 keys.
// Tried: a bulk copy for each row of 256 bytes, 18 cycles of the copy engine each (64 x 16,384 keys 280 to 362 us); rows on M, 8 to 16 of 16 of them empty (280 to 244 us); two or three
// parts to a resident block, for the slow SMs' sake (131,072 keys 99 to 102 and 107 us: as many more parts to join); a warp for every 8 rows of a shared stage (gated 113 to 115 us).
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

template <int D, int NQ, int KG, int DG, int S> struct PagedShape {
    static constexpr int THREADS = 32 * KG * DG, ROWS = 8 * NQ, UNIT = 16 * KG;
    static constexpr int PITCH = D * 2 + 16;                                    // bytes of a row in shared memory: eight rows' chunks in different banks
    static constexpr int STAGE = 2 * 16 * PITCH;                                // keys and values of 16 keys
    static constexpr int TURNS = NQ > 2 ? 2 : 1;                                // a key group's output goes through the stage it used last, in as many turns
    static constexpr int RING = KG * S * STAGE, STATS = KG * ROWS * 8, TABLES = KG * DG * 256, HALVES = DG > 1 ? KG * DG * NQ * 512 : 0;
    static constexpr int SMEM = RING + STATS + TABLES + HALVES;
    static_assert(ROWS * D * 4 / TURNS <= STAGE && (D / 16 / DG) % (KG * TURNS) == 0, "the key groups share the dimensions of an output out");
    static_assert(KG > 1 && 2 * KG <= 15, "named barriers: one for a key group's stages, one for its halves of scores");
};

template <int D, int NQ, int KG, int DG, int S>
__global__ void __launch_bounds__(32 * KG * DG) paged_attention_kernel(const __grid_constant__ PagedParams p) {
    using Shape = PagedShape<D, NQ, KG, DG, S>;
    constexpr int ROWS = Shape::ROWS, UNIT = Shape::UNIT, STAGE = Shape::STAGE, PITCH = Shape::PITCH, CH = D / 8, MT = D / 16 / DG, WARPS = KG * DG;
    extern __shared__ __align__(128) uint8_t smem[];
    float2 *stat_sm = (float2 *)(smem + Shape::RING);
    longlong2 *row_sm = (longlong2 *)((uint8_t *)stat_sm + Shape::STATS);       // [warp][16]: bytes to the keys and values of the stage being asked for
    const gq_attention_args &a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, kg = warp / DG, dg = warp % DG, g = lane / 4, t = lane % 4;
    pdl_wait();
    pdl_trigger();

    float4 *half_sm = (float4 *)(row_sm + 16 * WARPS) + kg * DG * NQ * 32;             // [DG][NQ][lane]: scores over a dimension group's part of head_dim

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
                    for (int i = 0; i < COPIES / DG; ++i) {
                        const uint32_t row = (DG > 1 ? i * DG + dg : i) * PER;
                        cp_async16(dst + row * PITCH, k + (uint64_t)row * k_step);
                        cp_async16(dst + (16 + row) * PITCH, v + (uint64_t)row * v_step);
                    }
                } else {
                    bad = ok || seen <= 0 ? 0u : (1u << seen) - 1;
#pragma unroll 1
                    for (int i = dg; i < COPIES; i += DG) {
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
                for (int i = dg; i < COPIES; i += DG) {
                    const int row = i * PER;
                    const longlong2 at = rows_at[row + copy_row];
                    const bool is = real >> (row + copy_row) & 1;
                    cp_async16(dst + row * PITCH, k_head + at.x, is);
                    cp_async16(dst + (16 + row) * PITCH, v_head + at.y, is);
                }
            }
            if (bad && dg == 0 && lane == 0) atomicMax(p.status, GQ_DEV_BAD_SHAPE);
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

    // Transposed products: keys (or dimensions) on M, eight query rows on N, NQ times.  A lane holds, of a score tile, keys g and g + 8 of queries 2 t and 2 t + 1; of the
    // output, dimensions 16 i + g and 16 i + g + 8 of the same two queries.
    float o[NQ][MT][4], top[NQ][2], sum[NQ][2];
    uint32_t qf[NQ][MT][2];
    int lim[NQ][2], lim_first = 0;     // keys that this lane's queries see, and the tile's first row
    int slot = 0;
    // where this lane's row of an ldmatrix starts: keys (rows 0-7, 8-15 of one chunk, then of the next), values (transposed: two chunks of rows 0-7, then of 8-15)
    const uint32_t k_lane = (((lane >> 3) & 1) * 8 + (lane & 7)) * PITCH + (lane >> 4) * 16 + dg * MT * 32, v_lane = (16 + (lane >> 4) * 8 + (lane & 7)) * PITCH + ((lane >> 3) & 1) * 16 + dg * MT * 32;

    for (int it = 0;;) {
        const int unit0 = use.unit;         // this block's first unit of the segment
        const int rows = use.v.n * p.group, before = use.v.len - use.v.n + 1;
        lim_first = before + (unsigned)(use.tile * ROWS) / (unsigned)p.group;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[q][i][j] = 0.0f;
            const int row0 = use.tile * ROWS + q * 8;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[q][j] = -INFINITY;
                sum[q][j] = 0.0f;
                lim[q][j] = before + (unsigned)min(row0 + 2 * t + j, rows - 1) / (unsigned)p.group;
            }
            const int r = row0 + g, i = (unsigned)r / (unsigned)p.group;
            const uint32_t *src = (const uint32_t *)((const __nv_bfloat16 *)a.q + (use.v.tok0 + i) * a.q_strides[0] + (use.head * p.group + (r - i * p.group)) * a.q_strides[1] + dg * MT * 16) + t;
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int j = 0; j < 2; ++j) qf[q][x][j] = r < rows ? src[x * 8 + j * 4] : 0u;
        }
        for (const int end = min(use.units, use.unit + count - it); use.unit < end; ++use.unit) {
            cp_async_wait<S - 2>();
            if constexpr (DG > 1) asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * DG) : "memory");
            else __syncwarp();
            const uint32_t bad = (uint32_t)missing & 0xffffu;
            ask(slot == 0 ? S - 1 : slot - 1);

            // ---- scores of 16 keys ----
            const uint32_t stage = ring + slot * STAGE;
            float s[NQ][4] = {}, s2[NQ][4] = {};
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t kf[4];
                ldsm4(kf, stage + k_lane + i * 32);
#pragma unroll
                for (int q = 0; q < NQ; ++q) mma_bf16(i & 1 ? s2[q] : s[q], kf, qf[q][i][0], qf[q][i][1]);
            }
            if constexpr (DG > 1) {         // both halves add in the same order, and go on with the same scores
#pragma unroll
                for (int q = 0; q < NQ; ++q) half_sm[(dg * NQ + q) * 32 + lane] = make_float4(s[q][0] + s2[q][0], s[q][1] + s2[q][1], s[q][2] + s2[q][2], s[q][3] + s2[q][3]);
                asm volatile("bar.sync %0, %1;" ::"r"(1 + KG + kg), "n"(32 * DG) : "memory");
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const float4 a0 = half_sm[q * 32 + lane], a1 = half_sm[(NQ + q) * 32 + lane];
                    s[q][0] = a0.x; s[q][1] = a0.y; s[q][2] = a0.z; s[q][3] = a0.w;
                    s2[q][0] = a1.x; s2[q][1] = a1.y; s2[q][2] = a1.z; s2[q][3] = a1.w;
                }
            }
            const int key0 = (use.unit * KG + kg) * 16;
            const bool edge = key0 + 16 > lim_first || bad;        // a row of the tile does not see all of these keys, or a page is missing
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[q][j] = (s[q][j] + s2[q][j]) * p.scale2;
            if (edge) {
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = g + (j >> 1) * 8;
                        if (bad >> at & 1) s[q][j] = __int_as_float(0x7fc00000);
                        if (key0 + at >= lim[q][j & 1]) s[q][j] = -INFINITY;
                    }
            }
            // ---- probabilities, against a reference that follows the maximum from afar: a score may stand up to 2^8 over it, where nothing is near a limit or less exact, so that
            // after a segment's first keys no maximum is taken and nothing is scaled again ----
            bool higher = false;
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) higher |= s[q][j] > top[q][j & 1] + 8.0f;
            if (__any_sync(~0u, higher)) {
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    float keep[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float m = fmaxf(s[q][j], s[q][j + 2]);
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                        m = fmaxf(m, top[q][j]);
                        keep[j] = ex2(top[q][j] - (m == -INFINITY ? 0.0f : m));
                        top[q][j] = m;
                        sum[q][j] *= keep[j];
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[q][i][j] *= keep[j & 1];
                }
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[q][j] = ex2(s[q][j] - (top[q][j & 1] == -INFINITY ? 0.0f : top[q][j & 1]));
                    sum[q][j & 1] += s[q][j];
                }
            // ---- p v ----
            // Keys that some rows of the tile see and others do not: a masked probability of 0 would still make NaN of an infinite value, so these keys stay out of the MMA and are
            // added row by row.  There are fewer of them in all than new tokens in the tile.
            const bool split = edge && lim_first < use.keys;
            const int from = split ? max(lim_first - key0, 0) : 16;
            if (split) {
                const int to = min(use.keys - key0, 16);
                for (int x = from; x < to; ++x) {
                    const int owner = (x & 7) * 4 + t;
                    const __nv_bfloat16 *v = (const __nv_bfloat16 *)(smem + (stage - smem_u32(smem)) + (16 + x) * PITCH) + dg * MT * 16 + g;
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        const float pa = __shfl_sync(~0u, x & 8 ? s[q][2] : s[q][0], owner), pb = __shfl_sync(~0u, x & 8 ? s[q][3] : s[q][1], owner);
                        const bool see_a = key0 + x < lim[q][0], see_b = key0 + x < lim[q][1];
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float val = __bfloat162float(v[i * 16 + j * 8]);
                                if (see_a) o[q][i][2 * j] += pa * val;
                                if (see_b) o[q][i][2 * j + 1] += pb * val;
                            }
                    }
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (g + (j >> 1) * 8 >= from) s[q][j] = 0.0f;
            }
            // the probabilities of eight keys, turned over: queries on g, keys 2 t and 2 t + 1, as the B operand has them
            uint32_t big[NQ][2], small[NQ][2];
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    bf16_parts(s[q][2 * j], s[q][2 * j + 1], big[q][j], small[q][j]);
                    big[q][j] = transpose8(big[q][j]);
                    small[q][j] = transpose8(small[q][j]);
                }
            const uint32_t vm0 = (2 * t < from ? 0xffffu : 0u) | (2 * t + 1 < from ? 0xffff0000u : 0u), vm1 = (2 * t + 8 < from ? 0xffffu : 0u) | (2 * t + 9 < from ? 0xffff0000u : 0u);
            auto values = [&](bool masked) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    uint32_t vf[4];
                    ldsm4_t(vf, stage + v_lane + i * 32);
                    if (masked) { vf[0] &= vm0; vf[1] &= vm0; vf[2] &= vm1; vf[3] &= vm1; }
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        mma_bf16(o[q][i], vf, big[q][0], big[q][1]);
                        mma_bf16(o[q][i], vf, small[q][0], small[q][1]);
                    }
                }
            };
            if (split) values(true);
            else values(false);
            if (++slot == S) slot = 0;
            ++it;
        }

        // ---- the end of this block's part of a segment: key groups joined, from the first to the last ----
        constexpr int MINE = MT / KG, TURNS = Shape::TURNS;       // dimension tiles that a key group adds up, the turns of the exchange
        float sum_o[NQ][MINE][4], keep[NQ][KG][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) sum[q][j] += __shfl_xor_sync(~0u, sum[q][j], x);
                if (g == 0 && dg == 0) stat_sm[kg * ROWS + q * 8 + 2 * t + j] = make_float2(top[q][j], sum[q][j]);
            }
        const int used = (slot == 0 ? S - 1 : slot - 1) * STAGE;
        if constexpr (DG > 1) asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * DG) : "memory");      // nobody reads that stage any more
        else __syncwarp();
#pragma unroll
        for (int h = 0; h < TURNS; ++h) {
            constexpr int PART = MT / TURNS;
            float4 *box = (float4 *)(smem + kg * S * STAGE + used) + dg * NQ * PART * 32 + lane;
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    const float(&v)[4] = o[q][h * PART + i];
                    box[(q * PART + i) * 32] = make_float4(v[0], v[1], v[2], v[3]);
                }
            __syncthreads();
            if (h == 0) {
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 *st = stat_sm + q * 8 + 2 * t + j;
                        float m = -INFINITY;
                        for (int x = 0; x < KG; ++x) m = fmaxf(m, st[x * ROWS].x);
                        const float r = m == -INFINITY ? 0.0f : m;
                        top[q][j] = m;
                        sum[q][j] = 0.0f;
#pragma unroll
                        for (int x = 0; x < KG; ++x) {
                            keep[q][x][j] = ex2(st[x * ROWS].x - r);
                            sum[q][j] += st[x * ROWS].y * keep[q][x][j];
                        }
                    }
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int i = 0; i < MINE / TURNS; ++i) {
                    float(&v)[4] = sum_o[q][h * (MINE / TURNS) + i];
                    v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
                    for (int x = 0; x < KG; ++x) {
                        const float4 w = ((const float4 *)(smem + x * S * STAGE + used))[dg * NQ * PART * 32 + (q * PART + i * KG + kg) * 32 + lane];
                        v[0] += w.x * keep[q][x][0]; v[1] += w.y * keep[q][x][1]; v[2] += w.z * keep[q][x][0]; v[3] += w.w * keep[q][x][1];
                    }
                }
            __syncthreads();            // the next turn, or the next stage, comes to the same place
        }
        auto dim_of = [&](int i) { return ((i / (MINE / TURNS)) * (MT / TURNS) + (i % (MINE / TURNS)) * KG + kg + dg * MT) * 16 + g; };       // of sum_o[.][i][0], [1]; 8 more: of [2], [3]
        const bool whole = unit0 == 0 && use.unit == use.units;
        const int64_t part = 2 * (int64_t)blockIdx.x + (unit0 == 0);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int in_tile = q * 8 + 2 * t + j, r = use.tile * ROWS + in_tile;
                if (r >= rows) continue;
                if (whole) {
                    const int i0 = (unsigned)r / (unsigned)p.group;
                    const int64_t tok = use.v.tok0 + i0, h = use.head * p.group + (r - i0 * p.group);
                    __nv_bfloat16 *dst = (__nv_bfloat16 *)a.out + tok * a.out_strides[0] + h * a.out_strides[1];
                    const __nv_bfloat16 *gate = a.gate ? (const __nv_bfloat16 *)a.gate + tok * a.gate_strides[0] + h * a.gate_strides[1] : nullptr;
                    const float inv = sum[q][j] == 0.0f ? 0.0f : 1.0f / sum[q][j];
#pragma unroll
                    for (int i = 0; i < MINE; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int d = dim_of(i) + 8 * x;
                            float v = sum_o[q][i][2 * x + j] * inv;
                            if (gate && inv != 0.0f) v /= 1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[d]));        // no key: zeros, whatever the gate
                            dst[d] = __float2bfloat16_rn(v);
                        }
                } else {
                    const int64_t at = part * ROWS + in_tile;
                    if (g == 0 && kg == 0 && dg == 0) p.stats[at] = make_float2(top[q][j], sum[q][j]);
#pragma unroll
                    for (int i = 0; i < MINE; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) p.parts[at * D + dim_of(i) + 8 * x] = sum_o[q][i][2 * x + j];
                }
            }
        if (it == count) break;
        next_segment<ROWS, UNIT>(p, use);
    }
    cp_async_wait<0>();
}

// The segments that several blocks worked on: block c joins the one that starts in block c's range and ends behind it, each row by as many warps as there are, four parts of
// a warp in flight.  All but the parts themselves is found before the wait for the kernel that writes them.
constexpr int JOIN_WARPS = 16;
template <int D, int ROWS, int UNIT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_parts_kernel(const __grid_constant__ PagedParams p) {
    constexpr int V = D / 32;                                   // values to a lane
    __shared__ float box[JOIN_WARPS][D];
    __shared__ float2 box_stats[JOIN_WARPS];
    const gq_attention_args &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int64_t end = 0;        // the block of the segment's last unit
    bool joins;
    Cursor c;
    {
        const Line line = count_units<ROWS, UNIT>(p, lane);
        const Cut cut = cut_line(p, line.total);
        const int64_t w0 = cut.start(blockIdx.x), w1 = cut.start(blockIdx.x + 1);
        joins = w0 != w1;
        if (joins) {
            locate<ROWS, UNIT>(p, line, w1 - 1, lane, c);
            const int64_t first = w1 - 1 - c.unit;
            joins = first >= w0 && first + c.units != w1;
            if (joins) end = min(cut.block_of(first + c.units - 1), cut.blocks - 1);
        }
    }
    // Blocks without a segment wait too: what is launched behind this kernel waits for this one alone, so it has to end behind the one in front.
    pdl_wait();
    if (!joins) return;
    const int rows = min(ROWS, c.v.n * p.group - c.tile * ROWS), sets = max(JOIN_WARPS / rows, 1), set = warp / min(rows, JOIN_WARPS);
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
                if (gate && inv != 0.0f) v /= 1.0f + ex2(-1.4426950408889634f * __bfloat162float(gate[i * 32]));
                dst[i * 32] = __float2bfloat16_rn(v);
            }
        }
    }
}

}  // namespace gq
