// The operators beside the quantized layers of a decoder block: low-rank adapters of many requests beside a layer, norms and rotation of
// queries and keys with the store into a paged cache, attention over that cache.  C ABI in include/gq_b200.h.
#include <cuda_runtime.h>
#include <atomic>
#include <stdint.h>
#include "gq_host.h"
#include "gq_adapters.cuh"
#include "gq_heads.cuh"
#include "gq_paged.cuh"

using namespace gq;

// the largest status code a kernel of this unit reported since it was last read
__device__ int g_block_status;

cudaError_t gq::block_status_read(int *code, cudaStream_t s) { return cudaMemcpyFromSymbolAsync(code, g_block_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s); }
cudaError_t gq::block_status_clear(cudaStream_t s) {
    static const int zero = 0;
    return cudaMemcpyToSymbolAsync(g_block_status, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, s);
}

static bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
// the word's address on the current device, asked for once
static int status_word(int **p) {
    static std::atomic<int *> known[64];
    int dev = 0;
    GQ_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && (*p = known[dev].load(std::memory_order_acquire))) return GQ_OK;
    GQ_CUDA(cudaGetSymbolAddress((void **)p, g_block_status));
    if (dev < 64) known[dev].store(*p, std::memory_order_release);
    return GQ_OK;
}

// Launches a kernel that begins with griddepcontrol.wait while the kernel in front of it ends.
template <class... P, class... A> static cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, int threads, int smem, void *stream, A... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream; cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// blocks of a kernel that the current device holds at once; its shared memory is allowed on the way (asked once per device)
template <auto KERNEL> static int resident_blocks(int threads, int smem, int *blocks) {
    static std::atomic<int> known[64];
    int dev = 0, sms = 0, per_sm = 0;
    GQ_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && (*blocks = known[dev].load(std::memory_order_acquire))) return GQ_OK;
    GQ_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    GQ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    GQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERNEL, threads, smem));
    *blocks = sms * (per_sm < 1 ? 1 : per_sm);
    if (dev < 64) known[dev].store(*blocks, std::memory_order_release);
    return GQ_OK;
}

// ---- low-rank adapters -------------------------------------------------------------------------------

static int check_low_rank(const gq_low_rank_args *p, int64_t *n_total) {
    if (!p || p->M < 0 || p->M > 65535 * (int64_t)LR_ROWS || p->K <= 0 || p->K % GQ_QK || p->K > (1 << 24) || p->rank <= 0 || p->rank % 8 || p->n_adapters <= 0) return p ? GQ_ERR_SHAPE : GQ_ERR_ARG;
    if (p->rank > GQ_MAX_RANK || p->n_shards < 1 || p->n_shards > GQ_MAX_DEVICE_SHARDS) return GQ_ERR_LIMIT;
    *n_total = 0;
    for (int s = 0; s < p->n_shards; ++s) {
        if (p->n_outs[s] < 0 || p->n_outs[s] > INT32_MAX) return GQ_ERR_SHAPE;
        *n_total += p->n_outs[s];
    }
    return *n_total > INT32_MAX ? GQ_ERR_SHAPE : GQ_OK;
}
static int64_t up256(int64_t v) { return (v + 255) & ~(int64_t)255; }
static int ranks_of(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }
// How the inner products are cut: sixteens of ranks to a block, blocks that share a tile's adapters, parts of K (256 at least; the blocks of a cluster), blocks for all ranks.
// 148, 74, 296 and 444 are one, a half, two and three blocks to each of a B200's SMs.  Clusters are powers of two, of sixteen only while there are few: thirteen parts of 2,051 rows beside gate_up took 8 us more than eight, sixteen for each of seven adapters of
// rank 32 beside qkv 4 us more than eight and fewer ranks to a block; one row beside qkv is 0.3 us faster with sixteen.
struct LowRankCut {
    int ranks, groups, parts, turns;
};
static LowRankCut low_rank_cut(const gq_low_rank_args *p) {
    const int64_t tiles = (p->M + LR_ROWS - 1) / LR_ROWS;
    const int sixteens = p->n_shards * ((p->rank + 15) / 16);
    LowRankCut c{};
    int64_t most;
    if (tiles > 1) {             // chunks: 32 or 64 ranks to a block, three blocks to an SM; two for a tile in which requests meet
        c.ranks = sixteens <= 2 ? 2 : 4;
        c.groups = p->n_adapters > 1 ? 2 : 1;
        c.turns = (sixteens + c.ranks - 1) / c.ranks;
        most = std::min<int64_t>(16, 444 / (c.turns * tiles));
    } else {                     // decode: every adapter a block of its own, as many ranks to it as leave the GPU full
        c.groups = (int)std::min<int64_t>(std::min<int64_t>(p->M, LR_ROWS), p->n_adapters);
        for (int n = 4; n >= 1; --n) {
            c.turns = (sixteens + n - 1) / n;
            c.ranks = (sixteens + c.turns - 1) / c.turns;
            if (c.turns * c.groups * 8 >= 148) break;
        }
        most = c.turns * c.groups * 8 < 74 ? 16 : std::min<int64_t>(8, 296 / (c.turns * c.groups));
    }
    most = std::min<int64_t>(most, p->K / 256);
    for (c.parts = 1; c.parts * 2 <= most; c.parts *= 2) {}
    return c;
}
extern "C" int64_t gq_low_rank_workspace_bytes(const gq_low_rank_args *p) {
    int64_t n = 0;
    if (const int rc = check_low_rank(p, &n)) return rc;
    return n == 0 ? 0 : 2 * up256(p->M * p->n_shards * ranks_of(p->rank) * 2);
}
// the inner products, a cluster to the parts of K
template <auto KERNEL> static int low_rank_inner(const LowRankParams &q, dim3 grid, int smem, void *stream) {
    static std::atomic<uint64_t> allowed{0};         // devices that know of the shared memory and of more than the portable cluster
    int dev = 0;
    GQ_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !(allowed.load() >> dev & 1)) {
        if (smem) GQ_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        GQ_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (dev < 64) allowed.fetch_or((uint64_t)1 << dev);
    }
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = q.parts; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(LR_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream; cfg.attrs = attr; cfg.numAttrs = 2;
    GQ_CUDA(cudaLaunchKernelEx(&cfg, KERNEL, q));
    GQ_LAUNCHED();
    return GQ_OK;
}
template <int KS> static int low_rank_outer(const LowRankParams &q, void *stream) {
    using Shape = ChunkShape<KS>;
    const bool few = q.M <= 64, own = q.n_adapters > 4;        // decode, and whether the rows of a tile may all have their own
    const int cols = few ? LR_OUTER_WARPS * 32 : Shape::COLS;
    int64_t blocks = 0;
    for (int s = 0; s < q.n_shards; ++s) blocks += (q.edges[s + 1] - q.edges[s] + cols - 1) / cols;
    if (few) {
        if (own) GQ_CUDA(launch_pdl(low_rank_few_kernel<KS, 4>, dim3((unsigned)blocks, (q.M + 3) / 4), LR_OUTER_WARPS * 32, 0, stream, q));
        else GQ_CUDA(launch_pdl(low_rank_few_kernel<KS, 16>, dim3((unsigned)blocks, (q.M + 15) / 16), LR_OUTER_WARPS * 32, 0, stream, q));
    } else {                      // as many walks down the rows as the GPU holds blocks, at least one for every block of columns
        int resident = 0;
        if (const int rc = resident_blocks<low_rank_chunk_kernel<KS>>(LR_THREADS, Shape::SMEM, &resident)) return rc;
        const int tiles = (q.M + Shape::ROWS - 1) / Shape::ROWS, walks = (int)std::max<int64_t>(1, std::min<int64_t>(tiles, resident / blocks)), per = (tiles + walks - 1) / walks;
        GQ_CUDA(launch_pdl(low_rank_chunk_kernel<KS>, dim3((unsigned)blocks, (tiles + per - 1) / per), LR_THREADS, Shape::SMEM, stream, q, per));
    }
    GQ_LAUNCHED();
    return GQ_OK;
}
extern "C" int gq_low_rank_add(const gq_low_rank_args *p, void *stream) {
    int64_t n = 0;
    if (const int rc = check_low_rank(p, &n)) return rc;
    if (p->M == 0 || n == 0) return GQ_OK;
    if (!p->base || !p->x || !p->a || !p->b || !p->scales || !p->ids || !p->out || (p->ids_bytes != 4 && p->ids_bytes != 8)) return GQ_ERR_ARG;
    if (!aligned(p->x, 16) || !aligned(p->a, 16) || !aligned(p->b, 16) || p->ldx % 8 || p->ldx < p->K || p->ld_base < n || p->ld_out < n || (p->out == p->base && p->M > 1 && p->ld_out != p->ld_base)) return GQ_ERR_ARG;
    const int64_t bytes = gq_low_rank_workspace_bytes(p);
    if (p->workspace_bytes < bytes || !p->workspace || !aligned(p->workspace, 256)) return GQ_ERR_WORKSPACE;
    int *status;
    if (const int rc = status_word(&status)) return rc;
    const int64_t tiles = (p->M + LR_ROWS - 1) / LR_ROWS;
    const LowRankCut cut = low_rank_cut(p);
    bool vec = aligned(p->base, 16) && aligned(p->out, 16) && p->ld_base % 8 == 0 && p->ld_out % 8 == 0;
    LowRankParams q{(const __nv_bfloat16 *)p->base, (const __nv_bfloat16 *)p->x, (const __nv_bfloat16 *)p->a, (const __nv_bfloat16 *)p->b, p->scales, p->ids,
                    (__nv_bfloat16 *)p->out, (__nv_bfloat16 *)p->workspace, (__nv_bfloat16 *)((uint8_t *)p->workspace + bytes / 2), status, p->ld_base, p->ldx, p->ld_out, n, {0},
                    (int)p->M, (int)p->K, p->n_shards, p->n_adapters, p->rank, ranks_of(p->rank), cut.parts, p->ids_bytes == 8, cut.groups, 0};
    for (int s = 0; s < p->n_shards; ++s) {
        q.edges[s + 1] = q.edges[s] + p->n_outs[s];
        vec = vec && q.edges[s] % 8 == 0;
    }
    q.vec = vec;
    const dim3 inner(cut.parts, (unsigned)tiles, cut.groups * cut.turns);
    int rc;
    if (tiles > 1)
        rc = cut.ranks == 2 ? low_rank_inner<low_rank_inner_chunk_kernel<32>>(q, inner, InnerShape<32>::SMEM, stream) : low_rank_inner<low_rank_inner_chunk_kernel<64>>(q, inner, InnerShape<64>::SMEM, stream);
    else
        rc = cut.ranks == 1 ? low_rank_inner<low_rank_inner_kernel<1>>(q, inner, 0, stream) : cut.ranks == 2 ? low_rank_inner<low_rank_inner_kernel<2>>(q, inner, 0, stream)
             : cut.ranks == 3 ? low_rank_inner<low_rank_inner_kernel<3>>(q, inner, 0, stream) : low_rank_inner<low_rank_inner_kernel<4>>(q, inner, 0, stream);
    if (rc) return rc;
    switch (q.ranks) {
        case 16: return low_rank_outer<1>(q, stream);
        case 32: return low_rank_outer<2>(q, stream);
        case 64: return low_rank_outer<4>(q, stream);
        default: return low_rank_outer<8>(q, stream);
    }
}

// ---- norms and rotation of heads ---------------------------------------------------------------------

extern "C" int gq_head_norm_rope(const gq_head_norm_args *p, void *stream) {
    if (!p) return GQ_ERR_ARG;
    const bool store = p->k_pages || p->v_pages || (p->slots && !p->k_out);       // a cache of no pages has no memory
    if (p->T < 0 || p->T > INT32_MAX || p->n_heads < 1 || p->n_kv_heads < 1 || p->head_dim < 8 || p->head_dim % 8 || p->rotary_dim < 0 || p->rotary_dim % 2 ||
        p->rotary_dim > p->head_dim) return GQ_ERR_SHAPE;
    if (p->head_dim > 512 || (int64_t)p->n_heads + 2 * (int64_t)p->n_kv_heads > 65535) return GQ_ERR_LIMIT;
    if (store && (p->page_size < 1 || p->n_pages < 0)) return GQ_ERR_SHAPE;
    if (p->T == 0) return GQ_OK;
    const int64_t width = ((int64_t)p->n_heads * (p->gated ? 2 : 1) + 2 * (int64_t)p->n_kv_heads) * p->head_dim;
    if (!p->qkv || !p->q_out || !p->positions || (p->rotary_dim && !p->inv_freq) || (p->positions_bytes != 4 && p->positions_bytes != 8) || p->ld_qkv < width) return GQ_ERR_ARG;
    if (!aligned(p->qkv, 16) || p->ld_qkv % 8 || !aligned(p->q_out, 16) || !aligned(p->q_norm, 16) || !aligned(p->k_norm, 16)) return GQ_ERR_ARG;
    if (store) {
        if ((p->n_pages && (!p->k_pages || !p->v_pages)) || !p->slots || (p->slots_bytes != 4 && p->slots_bytes != 8) || p->k_out || !aligned(p->k_pages, 16) || !aligned(p->v_pages, 16)) return GQ_ERR_ARG;
        for (int i = 0; i < 3; ++i)
            if (p->k_strides[i] < 0 || p->v_strides[i] < 0 || p->k_strides[i] % 8 || p->v_strides[i] % 8) return GQ_ERR_ARG;
    } else if (!p->k_out || !aligned(p->k_out, 16)) return GQ_ERR_ARG;
    int *status;
    if (const int rc = status_word(&status)) return rc;
    gq_head_norm_args a = *p;
    if (!store) a.slots = nullptr;                                           // what the kernels look at
    if (p->head_dim % 16 || (!p->interleaved && p->rotary_dim % 16)) {
        GQ_CUDA(launch_pdl(head_norm_any_kernel, dim3((unsigned)p->T, p->n_heads + (store ? 2 : 1) * p->n_kv_heads), 64, 0, stream, a, status));
    } else {
        int group = 1;                                                       // lanes of a head, a power of two
        while (group * 16 < p->head_dim) group *= 2;
        // Tokens to a block.  One each while that fills the GPU about once, then four, whose start (positions, turns, weights) is one.  As one / as four to a block, 40 / 8 heads of 128 with the store:
        // 256 tokens 4.2 / 7.7 us, 1,024 8.7 / 9.0, 1,536 12.2 / 13.1, 2,047 15.6 / 13.9, 4,096 32.6 / 27.6, 8,192 62 / 51; 24 / 4 gated heads of 256 1,536 13.0 / 14.9, 2,047 16.5 / 15.8, 8,192 66 / 57.
        const int batch = p->T >= 2048 ? HEAD_BATCH : 1;
        const unsigned blocks = (unsigned)((p->T + batch - 1) / batch);
        if (p->interleaved) GQ_CUDA(launch_pdl(head_norm_kernel<true>, dim3(blocks), HEAD_THREADS, 0, stream, a, batch, group, status));
        else GQ_CUDA(launch_pdl(head_norm_kernel<false>, dim3(blocks), HEAD_THREADS, 0, stream, a, batch, group, status));
    }
    GQ_LAUNCHED();
    return GQ_OK;
}

// ---- attention over pages ----------------------------------------------------------------------------

static int check_attention(const gq_attention_args *p) {
    if (!p) return GQ_ERR_ARG;
    if (p->T < 0 || p->T > INT32_MAX || p->n_seqs < 0 || p->n_seqs > INT32_MAX || p->table_width < 0 || p->n_pages < 0 || p->page_size < 1 || p->n_heads < 1 || p->n_kv_heads < 1 ||
        p->n_heads % p->n_kv_heads || (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)) return GQ_ERR_SHAPE;
    if (!p->q_starts && p->T && (p->n_seqs == 0 || p->T % p->n_seqs)) return GQ_ERR_SHAPE;
    if (p->n_heads > 65535 || p->T > (1 << 24) || p->T * (p->n_heads / p->n_kv_heads) >= (1 << 30) || p->table_width > (1 << 30) || p->table_width * p->page_size > (1 << 30)) return GQ_ERR_LIMIT;
    return GQ_OK;
}
// Rows of a tile, in eights: those of a sequence's tokens under one kv head, as far as the batch's average tells.  (16 x 4 tokens of 5 heads: 52 us as a warp for every 8 rows, 45 as three eights of one.)
// One width serves a whole batch, so a long chunk among decodes costs both: 1,024 tokens of one sequence and 63 decodes over 1,000 to 7,000 keys take 638 us in one call, 278 and 176 in two; with 16 tokens for
// 1,024 184 in one, 24 and 176 in two (heads 40 / 8 of 128).
static int row_eights(const gq_attention_args *p) {
    const int64_t tokens = p->n_seqs ? (p->T + p->n_seqs - 1) / p->n_seqs : 1, rows = tokens * (p->n_heads / p->n_kv_heads);
    return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4;
}
template <int D, int NQ, int KG, int DG, int S> static int attention(const gq_attention_args *p, int64_t *bytes, int *status, void *stream) {
    using Shape = PagedShape<D, NQ, KG, DG, S>;
    int blocks = 0;
    if (const int rc = resident_blocks<paged_attention_kernel<D, NQ, KG, DG, S>>(Shape::THREADS, Shape::SMEM, &blocks)) return rc;
    const int64_t slots = 2 * (int64_t)blocks * Shape::ROWS, at_parts = up256(slots * 8);
    *bytes = at_parts + slots * D * 4;
    if (!status) return GQ_OK;
    if (!p->workspace || !aligned(p->workspace, 256) || p->workspace_bytes < *bytes) return GQ_ERR_WORKSPACE;
    uint8_t *ws = (uint8_t *)p->workspace;
    uint32_t log2 = 0;
    while ((int64_t)1 << log2 < p->page_size) ++log2;
    PagedParams q{*p, status, (float2 *)ws, (float *)(ws + at_parts), p->n_heads / p->n_kv_heads, blocks, (int)(p->table_width * p->page_size),
                  p->q_starts ? 0 : (int)(p->T / p->n_seqs), p->page_size % 16 == 0 && p->k_strides[1] < (1 << 27) && p->v_strides[1] < (1 << 27),
                  (uint32_t)(((uint64_t)1 << (31 + log2)) / p->page_size + 1), 31 + log2, p->scale * 1.4426950408889634f};
    if (p->n_pages == 0) {       // every page is outside the cache: nothing is read, but addresses are formed
        q.a.k_pages = q.a.v_pages = p->q;
        for (int i = 0; i < 3; ++i) q.a.k_strides[i] = q.a.v_strides[i] = 0;
    }
    GQ_CUDA(launch_pdl(paged_attention_kernel<D, NQ, KG, DG, S>, dim3(blocks), Shape::THREADS, Shape::SMEM, stream, q));
    GQ_LAUNCHED();
    GQ_CUDA(launch_pdl(join_parts_kernel<D, Shape::ROWS, Shape::UNIT>, dim3(blocks), JOIN_WARPS * 32, 0, stream, q));
    GQ_LAUNCHED();
    return GQ_OK;
}
static int attention_by_shape(const gq_attention_args *p, int64_t *bytes, int *status, void *stream) {
    switch (p->head_dim * 8 + row_eights(p)) {
        case 64 * 8 + 1: return attention<64, 1, 4, 1, 3>(p, bytes, status, stream);
        case 64 * 8 + 2: return attention<64, 2, 4, 1, 3>(p, bytes, status, stream);
        case 64 * 8 + 3: return attention<64, 3, 2, 1, 3>(p, bytes, status, stream);
        case 64 * 8 + 4: return attention<64, 4, 2, 1, 3>(p, bytes, status, stream);
        case 128 * 8 + 1: return attention<128, 1, 4, 1, 3>(p, bytes, status, stream);
        case 128 * 8 + 2: return attention<128, 2, 4, 1, 3>(p, bytes, status, stream);
        case 128 * 8 + 3: return attention<128, 3, 4, 1, 3>(p, bytes, status, stream);
        case 128 * 8 + 4: return attention<128, 4, 2, 2, 3>(p, bytes, status, stream);
        case 256 * 8 + 1: return attention<256, 1, 4, 2, 3>(p, bytes, status, stream);
        case 256 * 8 + 2: return attention<256, 2, 4, 2, 3>(p, bytes, status, stream);
        case 256 * 8 + 3: return attention<256, 3, 4, 2, 3>(p, bytes, status, stream);
        default: return attention<256, 4, 4, 2, 3>(p, bytes, status, stream);
    }
}

extern "C" int64_t gq_attention_workspace_bytes(const gq_attention_args *p) {
    int64_t bytes = 0;
    if (const int rc = check_attention(p)) return rc;
    if (p->T == 0 || p->n_seqs == 0) return 0;
    const int rc = attention_by_shape(p, &bytes, nullptr, nullptr);
    return rc ? rc : bytes;
}
extern "C" int gq_paged_attention(const gq_attention_args *p, void *stream) {
    if (const int rc = check_attention(p)) return rc;
    if (p->T == 0 || p->n_seqs == 0) return GQ_OK;
    if (!p->q || !p->lens || !p->out || p->ld_table < p->table_width || (p->n_pages && (!p->k_pages || !p->v_pages)) || (p->table_width && !p->page_table)) return GQ_ERR_ARG;
    if (!aligned(p->q, 16) || !aligned(p->k_pages, 16) || !aligned(p->v_pages, 16)) return GQ_ERR_ARG;
    for (int i = 0; i < 3; ++i)
        if (p->k_strides[i] < 0 || p->v_strides[i] < 0 || p->k_strides[i] % 8 || p->v_strides[i] % 8 || (i < 2 && p->q_strides[i] % 8)) return GQ_ERR_ARG;
    int *status;
    if (const int rc = status_word(&status)) return rc;
    int64_t bytes;
    return attention_by_shape(p, &bytes, status, stream);
}
