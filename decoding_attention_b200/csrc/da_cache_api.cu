// C ABI of the operators around a quantised cache -- writing rows, reading them back, decode attention over them -- and
// of decode attention behind a shared prefix.
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/decoding_attn_b200.h"
#include "da_internal.h"
#include "da_kv_rows.h"
#include "da_prefix.h"
#include "da_stream.h"
#include "da_stream_plan.h"

namespace da {

int failf(int code, const char *fmt, ...) {
    char msg[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return report_error(code, msg);
}

int sm_count(int *out) {
    static std::atomic<int> known[64];  // 0: not asked yet
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64) {
        *out = known[dev].load(std::memory_order_relaxed);
        if (*out > 0) return DA_OK;
    }
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "device query: %s", cudaGetErrorString(e));
    if (dev < 64) known[dev].store(*out, std::memory_order_relaxed);
    return DA_OK;
}

StreamShape stream_shape(int dim, int kind, int group) {
    switch (dim) {
        case 64: return stream_shape_d64(kind, group);
        case 96: return stream_shape_d96(kind, group);
        case 128: return stream_shape_d128(kind, group);
        default: return stream_shape_d256(kind, group);
    }
}

namespace {
cudaError_t launch_stream(int dim, int kind, bool bf16, const StreamParams &p, cudaStream_t s) {
    switch (dim) {
        case 64: return launch_stream_d64(kind, bf16, p, s);
        case 96: return launch_stream_d96(kind, bf16, p, s);
        case 128: return launch_stream_d128(kind, bf16, p, s);
        case 256: return launch_stream_d256(kind, bf16, p, s);
        default: return cudaErrorInvalidValue;
    }
}

// Whether the tensor-core kernel for codes takes the call: 8-bit codes of head dims and groups that it has, in pages that a
// TMA box can fetch, and pieces that are worth its 128-key tiles.  With no more (sequence, KV head) pairs than CTA slots it
// is the faster one at any length (one sequence of 1 500 int8 keys, 8 heads: 8.6 us against 11.1); with more, a CTA works
// through several short sequences, and a piece costs it more (1 000 sequences of 65-130 keys, 32/8 heads: 93 us against 77 in
// int8, 111 against 68 in FP8; 256 of 1 000-2 000: 139 against 173 and 145 against 148).  The lengths are on the device: what
// the cache, or a row of the block table, holds a sequence is what there is to go by.  (A caller whose table is wider than
// its sequences passes the columns in use.)
bool on_codes_kernel(int dim, int kind, const StreamParams &p, int sms) {
    if ((kind != DA_KV_FP8_E4M3 && kind != DA_KV_INT8) || (dim != 96 && dim != 128) || p.group > codes_heads() || p.rows == 0) return false;
    if (p.block_table && p.page_shift < 4) return false;
    if ((int64_t)p.batch * p.head_k <= (int64_t)sms * codes_ctas()) return true;
    int64_t keys = p.rows / p.batch;
    if (p.block_table && ((int64_t)p.table_blocks << p.page_shift) < keys) keys = (int64_t)p.table_blocks << p.page_shift;
    return keys >= 512;
}
// Codes of a cache as [rows][head_k][dim] bytes.
int codes_map(const void *base, const StreamParams &p, int dim, CUtensorMap *out) {
    const uint64_t dims[3] = {(uint64_t)dim, (uint64_t)p.head_k, (uint64_t)p.rows};
    const uint64_t strides[2] = {(uint64_t)dim, (uint64_t)dim * p.head_k};
    const uint32_t box[3] = {128, 1, p.block_table && p.page_shift < 7 ? 1u << p.page_shift : 128u};
    return encode_tensor_map(base, 3, dims, strides, box, true, 2, out);
}
}  // namespace

// Launches the kernel that plan_stream chose; a DA_* status.
int run_stream(int dim, int kind, bool bf16, const StreamParams &p, cudaStream_t s) {
    cudaError_t e;
    if (p.on_codes) {
        int *status = nullptr;
        CUtensorMap tm_k, tm_v;
        int rc = xmerge_status_ptr(&status);
        if (rc == DA_OK) rc = codes_map(p.k, p, dim, &tm_k);
        if (rc == DA_OK) rc = codes_map(p.v, p, dim, &tm_v);
        if (rc != DA_OK) return rc;
        e = launch_codes(dim, kind, p, status, tm_k, tm_v, s);
    } else {
        e = launch_stream(dim, kind, bf16, p, s);
    }
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "decode kernel launch: %s", cudaGetErrorString(e));
    return DA_OK;
}

void plan_stream(int dim, int kind, int sms, StreamParams *p) {
    p->on_codes = on_codes_kernel(dim, kind, *p, sms) ? 1 : 0;
    if (p->on_codes) {
        const int slots = sms * codes_ctas();
        p->chunks = 1;
        p->spans = slots > p->head_k ? slots / p->head_k : 1;
        p->snap = 128;
        p->piece_cost = 128;  // a piece's start and end take about as long as a tile
        p->min_span = 256;
        return;
    }
    p->snap = 32;
    const StreamShape shape = stream_shape(dim, kind, p->group);
    p->chunks = (p->group + shape.heads - 1) / shape.heads;
    const int streams = p->head_k * p->chunks;
    p->head_warps = 1;
    while (p->head_warps < 8 && p->head_warps * 2 <= streams) p->head_warps *= 2;
    p->key_warps = 8 / p->head_warps;
    const int blocks = (streams + p->head_warps - 1) / p->head_warps;
    const int slots = sms * shape.ctas_per_sm;
    p->spans = slots > blocks ? slots / blocks : 1;
    // A piece of a sequence costs a CTA about as long as 64 keys of a warp, however short it is (its queries, the joining of
    // its warps, its output), and a span is longer than that.  With few sequences the spans' shortest length matters more
    // than their balance: half as much then.  (32 x 1 024-4 096 int4 keys, 32/2 heads: 25.0 us with a cost of 16, 24.0 with
    // 32, 22.9 with 64; 4 x 500-2 000, 32/8 heads: 13.3, 12.5 and 14.3.)
    const int cost = p->batch >= 16 ? 64 : 32;
    p->piece_cost = cost * p->key_warps;
    p->min_span = (cost + 32) * p->key_warps;
}

size_t stream_piece_bytes(const StreamParams &p, int dim) {
    return (size_t)p.spans * 2 * p.head_q * ((size_t)dim + 1) * sizeof(float);
}

// Conditions on the caches that every entry point of this file shares.
bool quantised_kind(int32_t kv_dtype) { return kv_dtype >= DA_KV_FP8_E4M3 && kv_dtype <= DA_KV_INT4; }
bool head_dim_supported(int64_t dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

namespace {

int check_rows_args(const da_kv_rows_args_t *a, bool write) {
    if (!a) return failf(DA_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof(*a))
        return failf(DA_ERR_INVALID_ARG, "struct_size %u != sizeof(da_kv_rows_args_t) %zu", a->struct_size, sizeof(*a));
    if (!quantised_kind(a->kv_dtype))
        return failf(DA_ERR_INVALID_ARG, "kv_dtype %d: 1 (FP8 e4m3), 2 (int8) or 3 (int4) expected", a->kv_dtype);
    if (a->x_dtype < DA_ROWS_FP16 || a->x_dtype > (write ? DA_ROWS_BF16 : DA_ROWS_FP32))
        return failf(DA_ERR_INVALID_ARG, "x_dtype %d: 0 (fp16)%s", a->x_dtype, write ? " or 1 (bf16) expected" : ", 1 (bf16) or 2 (fp32) expected");
    if (a->tokens < 0 || a->cache_rows < 0 || a->head_k <= 0) return failf(DA_ERR_INVALID_ARG, "tokens and cache_rows must not be negative, head_k must be positive");
    if (!head_dim_supported(a->dim)) return failf(DA_ERR_UNSUPPORTED, "unsupported dim %lld: 64, 96, 128 or 256", (long long)a->dim);
    if (a->tokens > 0 && (!a->k || !a->v)) return failf(DA_ERR_INVALID_ARG, "k and v must not be NULL");
    if (a->cache_rows > 0 && (!a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale))
        return failf(DA_ERR_INVALID_ARG, "k_cache, v_cache, k_scale and v_scale must not be NULL");
    if (a->head_k > INT32_MAX / 256 || a->tokens > INT32_MAX / a->head_k || a->cache_rows > INT64_MAX / 256 / a->head_k)
        return failf(DA_ERR_INVALID_ARG, "tokens * head_k must be below 2^31");
    if (!a->slots && a->tokens > a->cache_rows)
        return failf(DA_ERR_INVALID_ARG, "%lld tokens without slots do not fit %lld cache rows", (long long)a->tokens, (long long)a->cache_rows);
    if (((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache) & 15u)
        return failf(DA_ERR_INVALID_ARG, "k, v, k_cache and v_cache must be 16-byte aligned");
    if (((uintptr_t)a->k_scale | (uintptr_t)a->v_scale) & 3u || (uintptr_t)a->slots & 7u)
        return failf(DA_ERR_INVALID_ARG, "scales and slots must be aligned to their elements");
    const int64_t strides[2] = {a->k_row_stride, a->v_row_stride};
    for (int64_t s : strides)
        if (s != 0 && (s < a->head_k * a->dim || s % (a->x_dtype == DA_ROWS_FP32 ? 4 : 8) != 0))
            return failf(DA_ERR_INVALID_ARG, "row strides must be multiples of 16 bytes and cover a row");
    return DA_OK;
}

int run_rows(const da_kv_rows_args_t *a, bool write) {
    const int rc = check_rows_args(a, write);
    if (rc != DA_OK || a->tokens == 0) return rc;
    KvRowsParams p;
    memset(&p, 0, sizeof(p));
    p.k = a->k;
    p.v = a->v;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.slots = a->slots;
    p.k_row_stride = a->k_row_stride ? a->k_row_stride : a->head_k * a->dim;
    p.v_row_stride = a->v_row_stride ? a->v_row_stride : a->head_k * a->dim;
    p.cache_rows = a->cache_rows;
    p.rows = (uint32_t)(a->tokens * a->head_k);
    p.head_k = (int)a->head_k;
    p.by_heads = make_fast_div((uint32_t)a->head_k);
    const cudaError_t e = launch_kv_rows(p, (int)a->dim, a->x_dtype, a->kv_dtype, write, static_cast<cudaStream_t>(a->stream));
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "cache row kernel launch: %s", cudaGetErrorString(e));
    return DA_OK;
}

int check_quant_args(const da_quant_decode_args_t *a) {
    if (!a) return failf(DA_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof(*a))
        return failf(DA_ERR_INVALID_ARG, "struct_size %u != sizeof(da_quant_decode_args_t) %zu", a->struct_size, sizeof(*a));
    if (!quantised_kind(a->kv_dtype))
        return failf(DA_ERR_INVALID_ARG, "kv_dtype %d: 1 (FP8 e4m3), 2 (int8) or 3 (int4) expected", a->kv_dtype);
    if (!head_dim_supported(a->dim)) return failf(DA_ERR_UNSUPPORTED, "unsupported dim %lld: 64, 96, 128 or 256", (long long)a->dim);
    if (a->batch <= 0 || a->head_q <= 0 || a->head_k <= 0) return failf(DA_ERR_INVALID_ARG, "batch, head_q and head_k must be positive");
    if (a->head_q % a->head_k != 0)
        return failf(DA_ERR_INVALID_ARG, "head_q (%lld) must be a multiple of head_k (%lld)", (long long)a->head_q, (long long)a->head_k);
    if (a->batch > 65535 || a->head_q > 65535) return failf(DA_ERR_INVALID_ARG, "batch and head_q must be <= 65535");
    if (a->rows < 0 || a->rows > INT32_MAX) return failf(DA_ERR_INVALID_ARG, "rows must be in [0, 2^31)");
    if (!a->q || !a->o || !a->cu_seq_k) return failf(DA_ERR_INVALID_ARG, "q, o and cu_seq_k must not be NULL");
    if (a->rows > 0 && (!a->k || !a->v || !a->k_scale || !a->v_scale))
        return failf(DA_ERR_INVALID_ARG, "k, v, k_scale and v_scale must not be NULL");
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o | (uintptr_t)a->workspace) & 15u)
        return failf(DA_ERR_INVALID_ARG, "q, k, v, o and workspace must be 16-byte aligned");
    if (((uintptr_t)a->k_scale | (uintptr_t)a->v_scale | (uintptr_t)a->cu_seq_k | (uintptr_t)a->lse | (uintptr_t)a->block_table) & 3u)
        return failf(DA_ERR_INVALID_ARG, "scales, cu_seq_k, lse and block_table must be 4-byte aligned");
    const int64_t strides[2] = {a->q_row_stride, a->o_row_stride};
    for (int64_t s : strides)
        if (s != 0 && (s < a->head_q * a->dim || s % 8 != 0))
            return failf(DA_ERR_INVALID_ARG, "row strides must be multiples of 16 bytes and cover a row");
    if (a->block_table) {
        if (a->page_size < 1 || (a->page_size & (a->page_size - 1)) != 0)
            return failf(DA_ERR_UNSUPPORTED, "page_size %d: paged caches need a power of two", a->page_size);
        if (a->table_blocks <= 0 || a->table_blocks > INT32_MAX || a->block_table_stride < a->table_blocks)
            return failf(DA_ERR_INVALID_ARG, "table_blocks must be positive and block_table_stride cover them");
    } else if (a->page_size != 0 || a->table_blocks != 0 || a->block_table_stride != 0) {
        return failf(DA_ERR_INVALID_ARG, "page_size, table_blocks or block_table_stride given without a block_table");
    }
    return DA_OK;
}

void fill_quant(const da_quant_decode_args_t *a, int sms, StreamParams *p) {
    memset(p, 0, sizeof(*p));
    p->q = a->q;
    p->k = a->k;
    p->v = a->v;
    p->k_scale = a->k_scale;
    p->v_scale = a->v_scale;
    p->cu_seq_k = a->cu_seq_k;
    p->block_table = a->block_table;
    p->o = a->o;
    p->lse = a->lse;
    p->q_row_stride = a->q_row_stride ? a->q_row_stride : a->head_q * a->dim;
    p->o_row_stride = a->o_row_stride ? a->o_row_stride : a->head_q * a->dim;
    p->k_row_stride = p->v_row_stride = a->head_k * a->dim;
    p->rows = a->rows;
    p->table_stride = a->block_table_stride;
    p->table_blocks = (int)a->table_blocks;
    for (int ps = a->page_size; ps > 1; ps >>= 1) ++p->page_shift;
    p->batch = (int)a->batch;
    p->head_q = (int)a->head_q;
    p->head_k = (int)a->head_k;
    p->group = p->head_q / p->head_k;
    p->is_alibi = a->is_alibi ? 1 : 0;
    p->q_bf16 = a->is_bf16 ? 1 : 0;
    p->scale_log2 = (a->softmax_scale > 0.0f ? a->softmax_scale : (float)(1.0 / std::sqrt((double)a->dim))) * kLog2e;
    plan_stream((int)a->dim, a->kv_dtype, sms, p);
}

int check_prefix_args(const da_prefix_decode_args_t *a) {
    if (!a) return failf(DA_ERR_INVALID_ARG, "args is NULL");
    if (a->struct_size != sizeof(*a))
        return failf(DA_ERR_INVALID_ARG, "struct_size %u != sizeof(da_prefix_decode_args_t) %zu", a->struct_size, sizeof(*a));
    if (a->kv_dtype != DA_KV_SAME_AS_Q && !quantised_kind(a->kv_dtype))
        return failf(DA_ERR_INVALID_ARG, "kv_dtype %d: 0 (the type of q), 1 (FP8 e4m3), 2 (int8) or 3 (int4) expected", a->kv_dtype);
    const bool quant = a->kv_dtype != DA_KV_SAME_AS_Q;
    if (a->dim != 64 && a->dim != 96 && a->dim != 128) return failf(DA_ERR_UNSUPPORTED, "unsupported dim %lld: 64, 96 or 128", (long long)a->dim);
    if (a->batch <= 0 || a->head_q <= 0 || a->head_k <= 0) return failf(DA_ERR_INVALID_ARG, "batch, head_q and head_k must be positive");
    if (a->head_q % a->head_k != 0)
        return failf(DA_ERR_INVALID_ARG, "head_q (%lld) must be a multiple of head_k (%lld)", (long long)a->head_q, (long long)a->head_k);
    if (a->head_q / a->head_k > 128) return failf(DA_ERR_UNSUPPORTED, "more than 128 query heads per KV head");
    if (a->batch > 65535 || a->head_q > 65535) return failf(DA_ERR_INVALID_ARG, "batch and head_q must be <= 65535");
    if (a->prefix_len < 0 || a->prefix_len > (1 << 30)) return failf(DA_ERR_INVALID_ARG, "prefix_len must be in [0, 2^30]");
    // (rows of a KV head in 256s at most) x (keys in 128s) x KV heads are counted in 32 bits
    if ((a->batch * (a->head_q / a->head_k) / 64 + 2) * ((a->prefix_len + 127) / 128) * a->head_k > INT32_MAX)
        return failf(DA_ERR_UNSUPPORTED, "batch * head_q * prefix_len is too large");
    if (a->rows < 0 || a->rows > INT32_MAX || a->prefix_rows < 0 || a->prefix_rows > INT32_MAX)
        return failf(DA_ERR_INVALID_ARG, "rows and prefix_rows must be in [0, 2^31)");
    if (!a->q || !a->o || !a->cu_seq_k) return failf(DA_ERR_INVALID_ARG, "q, o and cu_seq_k must not be NULL");
    if (a->prefix_len > 0 && (!a->k_prefix || !a->v_prefix)) return failf(DA_ERR_INVALID_ARG, "k_prefix and v_prefix must not be NULL");
    if (a->rows > 0 && (!a->k || !a->v || (quant && (!a->k_scale || !a->v_scale))))
        return failf(DA_ERR_INVALID_ARG, "k, v and, for a quantised cache, k_scale and v_scale must not be NULL");
    if (!quant && (a->k_scale || a->v_scale)) return failf(DA_ERR_INVALID_ARG, "scales given for a cache that is not quantised");
    if (((uintptr_t)a->q | (uintptr_t)a->k_prefix | (uintptr_t)a->v_prefix | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->o |
         (uintptr_t)a->workspace) & 15u)
        return failf(DA_ERR_INVALID_ARG, "q, k_prefix, v_prefix, k, v, o and workspace must be 16-byte aligned");
    if (((uintptr_t)a->k_scale | (uintptr_t)a->v_scale | (uintptr_t)a->cu_seq_k | (uintptr_t)a->lse | (uintptr_t)a->block_table |
         (uintptr_t)a->prefix_table) & 3u)
        return failf(DA_ERR_INVALID_ARG, "scales, cu_seq_k, lse and tables must be 4-byte aligned");
    const int64_t strides[6] = {a->q_row_stride, a->o_row_stride, a->k_prefix_row_stride, a->v_prefix_row_stride, a->k_row_stride, a->v_row_stride};
    for (int i = 0; i < 6; ++i)
        if (strides[i] != 0 && (strides[i] < (i < 2 ? a->head_q : a->head_k) * a->dim || strides[i] % 8 != 0 || (i >= 4 && quant)))
            return failf(DA_ERR_INVALID_ARG, "row strides must be multiples of 16 bytes and cover a row; a quantised cache is packed");
    if (a->prefix_table) {
        if (a->prefix_page_size < 16 || (a->prefix_page_size & (a->prefix_page_size - 1)) != 0)
            return failf(DA_ERR_UNSUPPORTED, "prefix_page_size %d: a paged prefix needs a power of two >= 16", a->prefix_page_size);
    } else {
        if (a->prefix_page_size != 0) return failf(DA_ERR_INVALID_ARG, "prefix_page_size given without a prefix_table");
        if (a->prefix_len > a->prefix_rows) return failf(DA_ERR_INVALID_ARG, "prefix_len exceeds prefix_rows");
    }
    if (a->block_table) {
        if (a->page_size < 1 || (a->page_size & (a->page_size - 1)) != 0)
            return failf(DA_ERR_UNSUPPORTED, "page_size %d: paged caches need a power of two", a->page_size);
        if (a->table_blocks <= 0 || a->table_blocks > INT32_MAX || a->block_table_stride < a->table_blocks)
            return failf(DA_ERR_INVALID_ARG, "table_blocks must be positive and block_table_stride cover them");
    } else if (a->page_size != 0 || a->table_blocks != 0 || a->block_table_stride != 0) {
        return failf(DA_ERR_INVALID_ARG, "page_size, table_blocks or block_table_stride given without a block_table");
    }
    return DA_OK;
}

PrefixGrid plan_prefix(int sms, int batch, int head_k, int group, int prefix_len) {
    PrefixGrid g;
    memset(&g, 0, sizeof(g));
    g.tile_seqs = 128 / group < batch ? 128 / group : batch;
    g.row_tiles = (batch + g.tile_seqs - 1) / g.tile_seqs;
    g.pairs = (g.row_tiles + 1) / 2;
    g.key_tiles = (prefix_len + 127) / 128;
    const int64_t total = (int64_t)head_k * g.pairs * g.key_tiles;
    g.total = (int)total;
    g.sms = sms;
    g.cta_tiles = (int)((total + sms - 1) / sms);
    g.ctas = (int)((total + g.cta_tiles - 1) / g.cta_tiles);
    // parts of a unit: the runs that touch it, twice where its streams share one row tile
    const int runs = (g.key_tiles + g.cta_tiles - 2) / g.cta_tiles + 1;
    g.max_parts = runs * (g.row_tiles % 2 ? 2 : 1);
    return g;
}

// What a key of the sequences' own costs an SM, in 1/65536 of a key tile of the prefix; 0 where the prefix does not fill the
// SMs anyway.  Measured: a key tile of two row tiles takes an SM 2.6 us at dim 128, an SM alone streams 54 GB/s of 16-bit
// rows, and codes take 7 (int8), 8 (FP8) or 9 ns (int4) for a key and KV head of 128 columns and eight query heads.
int own_cost(const StreamParams &s, const PrefixGrid &g, int dim, int kind) {
    if (g.total < 2 * g.sms) return 0;
    const double tile = (dim <= 64 ? 1800.0 : 2600.0) * g.row_tiles / (2 * g.pairs);
    const double bytes = kind == DA_KV_SAME_AS_Q ? 4.0 * dim : (kind == DA_KV_INT4 ? 1.0 : 2.0) * dim + 8;
    const double memory = bytes / 54.0, work = (kind == DA_KV_FP8_E4M3 ? 8.0 : (kind == DA_KV_INT4 ? 9.0 : 7.0)) * ((s.group + 7) / 8) * dim / 128;
    const double share = s.head_k * (memory > work ? memory : work) / tile * 65536.0;
    return share < 1.0 ? 1 : (share > 1e9 ? 1000000000 : (int)share);
}

struct PrefixPlan {
    PrefixGrid grid;
    size_t parts, own, pieces;  // floats of each area of the workspace, a multiple of 4
    size_t bytes() const { return (parts + own + pieces) * sizeof(float); }
};

PrefixPlan fill_prefix(const da_prefix_decode_args_t *a, int sms, StreamParams *s) {
    da_quant_decode_args_t d;  // the sequences' own keys are the other entry point's problem
    memset(&d, 0, sizeof(d));
    d.is_bf16 = a->is_bf16;
    d.is_alibi = a->is_alibi;
    d.kv_dtype = a->kv_dtype;
    d.q = a->q;
    d.k = a->k;
    d.v = a->v;
    d.k_scale = a->k_scale;
    d.v_scale = a->v_scale;
    d.o = a->o;
    d.lse = a->lse;
    d.cu_seq_k = a->cu_seq_k;
    d.rows = a->rows;
    d.batch = a->batch;
    d.head_q = a->head_q;
    d.head_k = a->head_k;
    d.dim = a->dim;
    d.q_row_stride = a->q_row_stride;
    d.o_row_stride = a->o_row_stride;
    d.block_table = a->block_table;
    d.block_table_stride = a->block_table_stride;
    d.table_blocks = a->table_blocks;
    d.page_size = a->page_size;
    d.softmax_scale = a->softmax_scale;
    fill_quant(&d, sms, s);
    if (a->k_row_stride) s->k_row_stride = a->k_row_stride;
    if (a->v_row_stride) s->v_row_stride = a->v_row_stride;
    const size_t rows = (size_t)a->batch * a->head_q, row = (size_t)a->dim + 1;
    PrefixPlan plan;
    memset(&plan, 0, sizeof(plan));
    if (a->prefix_len > 0) {
        plan.grid = plan_prefix(sms, s->batch, s->head_k, s->group, (int)a->prefix_len);
        plan.grid.own_cost = own_cost(*s, plan.grid, (int)a->dim, a->kv_dtype);
        plan.grid.most_tiles = (int)(((int64_t)plan.grid.total * 4 + sms - 1) / sms);
        plan.grid.by_sms = ~0ull / ((unsigned long long)sms << 16) + 1;
        if (plan.grid.own_cost) s->beside = plan.grid;
        plan.parts = ((size_t)plan.grid.max_parts * rows * row + 3) / 4 * 4;
        plan.own = (rows * row + 3) / 4 * 4;
    }
    plan.pieces = stream_piece_bytes(*s, (int)a->dim) / sizeof(float);
    return plan;
}

// Row maps of a prefix: K or V as [rows][head_k][dim], 64 columns of a box of rows.
int prefix_map(const void *base, int64_t rows, int64_t row_stride, int box_rows, const da_prefix_decode_args_t *a, CUtensorMap *out) {
    const uint64_t dims[3] = {(uint64_t)a->dim, (uint64_t)a->head_k, (uint64_t)rows};
    const uint64_t strides[2] = {(uint64_t)a->dim * 2, (uint64_t)row_stride * 2};
    const uint32_t box[3] = {64, 1, (uint32_t)box_rows};
    return encode_tensor_map(base, 3, dims, strides, box, true, a->is_bf16 ? 1 : 0, out);
}

}  // namespace
}  // namespace da

using namespace da;

extern "C" {

int da_kv_cache_write(const da_kv_rows_args_t *args) { return run_rows(args, true); }
int da_kv_cache_read(const da_kv_rows_args_t *args) { return run_rows(args, false); }

size_t da_quant_decode_workspace_bytes(const da_quant_decode_args_t *a) {
    int sms = 0;
    if (check_quant_args(a) != DA_OK || sm_count(&sms) != DA_OK) return 0;
    StreamParams p;
    fill_quant(a, sms, &p);
    return stream_piece_bytes(p, (int)a->dim);
}

int da_quant_decode_fwd(const da_quant_decode_args_t *a) {
    int sms = 0;
    int rc = check_quant_args(a);
    if (rc == DA_OK) rc = sm_count(&sms);
    if (rc != DA_OK) return rc;
    StreamMergeParams m;
    memset(&m, 0, sizeof(m));
    fill_quant(a, sms, &m.s);
    const size_t need = stream_piece_bytes(m.s, (int)a->dim);
    if (!a->workspace || a->workspace_bytes < need)
        return failf(DA_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", a->workspace ? a->workspace_bytes : (size_t)0, need);
    m.s.part_o = static_cast<float *>(a->workspace);
    m.s.part_lse = m.s.part_o + (size_t)m.s.spans * 2 * m.s.head_q * a->dim;
    m.dim = (int)a->dim;
    m.sms = sms;
    m.o = a->o;
    m.lse = a->lse;
    cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    rc = run_stream(m.dim, a->kv_dtype, a->is_bf16 != 0, m.s, stream);
    if (rc != DA_OK) return rc;
    const cudaError_t e = launch_stream_merge(m, stream);
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "decode kernel launch: %s", cudaGetErrorString(e));
    return DA_OK;
}

size_t da_prefix_decode_workspace_bytes(const da_prefix_decode_args_t *a) {
    int sms = 0;
    if (check_prefix_args(a) != DA_OK || sm_count(&sms) != DA_OK) return 0;
    StreamParams s;
    return fill_prefix(a, sms, &s).bytes();
}

int da_prefix_decode_fwd(const da_prefix_decode_args_t *a) {
    int sms = 0;
    int rc = check_prefix_args(a);
    if (rc == DA_OK) rc = sm_count(&sms);
    if (rc != DA_OK) return rc;
    StreamMergeParams m;
    memset(&m, 0, sizeof(m));
    const PrefixPlan plan = fill_prefix(a, sms, &m.s);
    if (!a->workspace || a->workspace_bytes < plan.bytes())
        return failf(DA_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", a->workspace ? a->workspace_bytes : (size_t)0, plan.bytes());
    float *parts = static_cast<float *>(a->workspace);
    const size_t rows = (size_t)a->batch * a->head_q;
    m.s.part_o = parts + plan.parts + plan.own;
    m.s.part_lse = m.s.part_o + (size_t)m.s.spans * 2 * m.s.head_q * a->dim;
    m.dim = (int)a->dim;
    m.sms = sms;
    m.o = a->o;
    m.lse = a->lse;
    cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    cudaError_t e = cudaSuccess;
    if (a->prefix_len > 0) {
        PrefixParams p;
        memset(&p, 0, sizeof(p));
        p.grid = plan.grid;
        p.k = a->k_prefix;
        p.v = a->v_prefix;
        p.table = a->prefix_table;
        p.k_row_stride = a->k_prefix_row_stride ? a->k_prefix_row_stride : a->head_k * a->dim;
        p.v_row_stride = a->v_prefix_row_stride ? a->v_prefix_row_stride : a->head_k * a->dim;
        p.rows = a->prefix_table ? a->prefix_rows : a->prefix_len;
        for (int ps = a->prefix_page_size; ps > 1; ps >>= 1) ++p.page_shift;
        p.prefix_len = (int)a->prefix_len;
        p.batch = m.s.batch;
        p.head_q = m.s.head_q;
        p.head_k = m.s.head_k;
        p.group = m.s.group;
        p.dim = (int)a->dim;
        p.cu_seq_k = a->cu_seq_k;
        p.is_alibi = m.s.is_alibi;
        p.scale_log2 = m.s.scale_log2;
        p.part_o = parts;
        p.part_lse = parts + (size_t)plan.grid.max_parts * rows * a->dim;
        rc = xmerge_status_ptr(&p.status);
        CUtensorMap tm_q, tm_k, tm_v;
        const int box = a->prefix_table && a->prefix_page_size < 128 ? a->prefix_page_size : 128;
        const uint64_t qd[3] = {(uint64_t)a->dim, (uint64_t)a->head_q, (uint64_t)a->batch};
        const uint64_t qs[2] = {(uint64_t)a->dim * 2, (uint64_t)m.s.q_row_stride * 2};
        const uint32_t qb[3] = {64, (uint32_t)p.group, (uint32_t)plan.grid.tile_seqs};
        if (rc == DA_OK) rc = encode_tensor_map(a->q, 3, qd, qs, qb, true, a->is_bf16 ? 1 : 0, &tm_q);
        if (rc == DA_OK) rc = prefix_map(p.k, p.rows, p.k_row_stride, box, a, &tm_k);
        if (rc == DA_OK) rc = prefix_map(p.v, p.rows, p.v_row_stride, box, a, &tm_v);
        if (rc != DA_OK) return rc;
        e = launch_prefix(a->is_bf16 != 0, p, tm_q, tm_k, tm_v, stream);
        m.prefix_o = p.part_o;
        m.prefix_lse = p.part_lse;
        m.prefix = plan.grid;
        m.s.o = nullptr;
        m.s.lse = nullptr;
        m.s.own_o = parts + plan.parts;
        m.s.own_lse = m.s.own_o + rows * a->dim;
        m.s.chained = 1;
    }
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "shared-prefix kernel launch: %s", cudaGetErrorString(e));
    rc = run_stream(m.dim, a->kv_dtype, a->is_bf16 != 0, m.s, stream);
    if (rc != DA_OK) return rc;
    e = launch_stream_merge(m, stream);
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "shared-prefix kernel launch: %s", cudaGetErrorString(e));
    return DA_OK;
}

}  // extern "C"
