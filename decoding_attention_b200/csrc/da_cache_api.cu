// C ABI of the operators around a quantised cache: writing rows, reading them back, decode attention over them.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/decoding_attn_b200.h"
#include "da_internal.h"
#include "da_kv_rows.h"
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
    static int known[64];  // 0: not asked yet (every thread would store the same value)
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64 && known[dev] > 0) {
        *out = known[dev];
        return DA_OK;
    }
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "device query: %s", cudaGetErrorString(e));
    if (dev < 64) known[dev] = *out;
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

cudaError_t launch_stream(int dim, int kind, bool bf16, const StreamParams &p, cudaStream_t s, bool overlap) {
    switch (dim) {
        case 64: return launch_stream_d64(kind, bf16, p, s, overlap);
        case 96: return launch_stream_d96(kind, bf16, p, s, overlap);
        case 128: return launch_stream_d128(kind, bf16, p, s, overlap);
        case 256: return launch_stream_d256(kind, bf16, p, s, overlap);
        default: return cudaErrorInvalidValue;
    }
}

void plan_stream(int dim, int kind, int sms, StreamParams *p) {
    const StreamShape shape = stream_shape(dim, kind, p->group);
    p->chunks = (p->group + shape.heads - 1) / shape.heads;
    const int streams = p->head_k * p->chunks;
    p->head_warps = 1;
    while (p->head_warps < 8 && p->head_warps * 2 <= streams) p->head_warps *= 2;
    p->key_warps = 8 / p->head_warps;
    const int blocks = (streams + p->head_warps - 1) / p->head_warps;
    const int slots = sms * shape.ctas_per_sm;
    p->spans = slots > blocks ? slots / blocks : 1;
    // A warp runs at least two or four tiles: below that its start costs more than its keys.
    p->min_span = p->key_warps * 32 > 64 ? p->key_warps * 32 : 64;
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
    if (a->head_k > INT32_MAX / 256 || a->tokens * a->head_k > (int64_t)INT32_MAX || a->cache_rows > INT64_MAX / 256 / a->head_k)
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
    m.o = a->o;
    m.lse = a->lse;
    cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    cudaError_t e = launch_stream(m.dim, a->kv_dtype, a->is_bf16 != 0, m.s, stream, false);
    if (e == cudaSuccess) e = launch_stream_merge(m, stream, true);
    if (e != cudaSuccess) return failf(DA_ERR_CUDA, "decode kernel launch: %s", cudaGetErrorString(e));
    return DA_OK;
}

}  // extern "C"
