// Launch parameters of the key-stream decode kernels (da_stream_kernel.cuh) and of the merge behind them.
#pragma once

#include <climits>

#include <cuda_runtime.h>

#include <cstdint>

#include "da_prefix.h"

namespace da {

// The batch's work is an axis on which sequence b takes piece_cost + len(b) units: what a piece costs however short it is,
// in keys, then its keys.  The axis is cut into `spans` equal spans, one per CTA (and head block); a cut falls on a multiple
// of `snap` keys of its sequence.
constexpr int kSpanUnits = 32;  // spans are multiples of this

struct StreamParams {
    const void *q;                 // [batch, head_q, dim]
    const void *k, *v;             // [rows, head_k, dim] elements or codes
    const float *k_scale, *v_scale;  // [rows, head_k], quantised caches only
    const int *cu_seq_k;           // [batch + 1]
    const int *block_table;        // optional [batch, table_stride]
    void *o;                       // [batch, head_q, dim]; NULL: whole sequences go to own_o / own_lse
    float *lse;                    // optional [batch, head_q]
    float *own_o, *own_lse;        // fp32 results of sequences that one CTA holds, when o is NULL
    float *part_o, *part_lse;      // pieces of the others [spans][2][head_q][dim], [spans][2][head_q]
    long long q_row_stride, k_row_stride, v_row_stride, o_row_stride;  // in elements
    long long rows;                // rows of k and v (pages * page_size); rows outside are masked
    long long table_stride;
    int table_blocks;              // pages of a table row
    int page_shift;
    int batch, head_q, head_k, group;
    int chunks;                    // warps that share a KV head (each has up to 8 NT of its query heads)
    int head_warps, key_warps;     // a CTA's eight warps: so many (KV head, chunk) streams x so many parts of the keys
    int spans, min_span;           // CTAs along the axis; no span is shorter than min_span units
    int piece_cost, snap;          // piece_cost + snap <= min_span: a sequence has keys in its first or second span
    int is_alibi, q_bf16;
    float scale_log2;              // softmax scale * log2(e)
    // Launched while the prefix kernel still runs: the grid then ends only after that one has, so that whoever waits for
    // this grid may read the other's results too (stays_for_prefix).
    int chained;
    PrefixGrid beside;             // the prefix kernel's, if the SMs are shared with it (own_cost)
    int on_codes;                  // host side: the kernel that takes the call (plan_stream)
};

// kind: 0 the type of q, 1 FP8 e4m3, 2 int8, 3 int4.
struct StreamShape {
    int heads;         // query heads of a warp (8 NT)
    int ctas_per_sm;
};
StreamShape stream_shape_d64(int kind, int group);
StreamShape stream_shape_d96(int kind, int group);
StreamShape stream_shape_d128(int kind, int group);
StreamShape stream_shape_d256(int kind, int group);
cudaError_t launch_stream_d64(int kind, bool bf16, const StreamParams &p, cudaStream_t s);
cudaError_t launch_stream_d96(int kind, bool bf16, const StreamParams &p, cudaStream_t s);
cudaError_t launch_stream_d128(int kind, bool bf16, const StreamParams &p, cudaStream_t s);
cudaError_t launch_stream_d256(int kind, bool bf16, const StreamParams &p, cudaStream_t s);

// The tensor-core kernel for 8-bit codes (da_codes_sm100.cu), head dims 96 and 128, groups of at most codes_heads() query
// heads: p.spans spans, cuts at multiples of 128 keys, pages of 16 keys or more.  kind: 1 FP8 e4m3, 2 int8.  tm_k, tm_v:
// [rows][head_k][dim] bytes, box {128, 1, 128 keys or a shorter page} with the 128-byte swizzle; rows beyond p.rows come as zeros.
int codes_heads();
int codes_ctas();  // per SM
cudaError_t launch_codes(int dim, int kind, const StreamParams &p, int *status, const CUtensorMap &tm_k, const CUtensorMap &tm_v,
                         cudaStream_t s);

// o = softmax-weighted sum of a row's pieces: those of the key stream and, with a shared prefix, its parts.
struct StreamMergeParams {
    StreamParams s;
    const float *prefix_o, *prefix_lse;  // [max_parts][batch][head_q][dim], [max_parts][batch][head_q]; NULL: no prefix
    PrefixGrid prefix;
    int dim, sms;
    void *o;      // [batch, head_q, dim], rows s.o_row_stride apart
    float *lse;   // optional [batch, head_q]
};
cudaError_t launch_stream_merge(const StreamMergeParams &p, cudaStream_t s);

// The cut of the axis into spans, the same in the stream kernel and in the merge.
struct SpanPlan {
    long long units;  // of a span
    long long total;  // of the batch
    int first;        // cu_seq_k[0]
    int cost, snap;
};
#ifdef __CUDACC__
// a / b of positions on the axis, which nearly always fit 32 bits (a 64-bit division takes ten times as long).
__device__ __forceinline__ long long axis_div(long long a, long long b) {
    return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
__device__ __forceinline__ SpanPlan span_plan(const StreamParams &p) {
    SpanPlan s;
    s.first = p.cu_seq_k[0];
    s.cost = p.piece_cost;
    s.snap = p.snap;  // a power of two
    const long long keys = (long long)p.cu_seq_k[p.batch] - s.first;
    s.total = (keys > 0 ? keys : 0) + (long long)p.batch * s.cost;
    int spans = p.spans;
    if (p.beside.own_cost) {
        // As many spans as the SMs that the prefix leaves free take in whole waves.
        const int run = prefix_run(p.beside, keys > 0 ? keys : 0);
        const unsigned sms = p.beside.sms, left = sms - ((unsigned)p.beside.total + run - 1) / (unsigned)run;
        if (run > p.beside.cta_tiles && left > 0) spans = (int)((unsigned)spans * (sms / left * left) / sms);
        if (spans < 1) spans = 1;
    }
    long long units = axis_div(s.total + spans - 1, spans);
    if (units < p.min_span) units = p.min_span;
    s.units = (units + kSpanUnits - 1) / kSpanUnits * kSpanUnits;
    return s;
}
// Keys of sequence b, which starts at cu.  (The bound keeps the indices of a tile behind the last key inside 32 bits; a
// cache has fewer rows.)
__device__ __forceinline__ int sequence_keys(const StreamParams &p, int b, int cu) {
    const long long n = (long long)p.cu_seq_k[b + 1] - cu;
    return n < 0 ? 0 : (n > INT_MAX - 1024 ? INT_MAX - 1024 : (int)n);
}
// Whether this block waits for the prefix kernel before it ends.  One block is enough for the grid's end to come after; where
// the SMs are shared with the prefix the others make room for those that have not started.
__device__ __forceinline__ bool stays_for_prefix(const StreamParams &p) {
    return p.chained && (!p.beside.own_cost || (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1));
}
// Where sequence b, whose keys start at cu, begins on the axis.
__device__ __forceinline__ long long axis_start(const SpanPlan &s, int b, int cu) {
    return (long long)cu - s.first + (long long)b * s.cost;
}
// Keys [begin, end) that span i has of a sequence of `len` keys that begins at `start` on the axis.
__device__ __forceinline__ void span_piece(const SpanPlan &s, long long i, long long start, int len, int &begin, int &end) {
    const long long lo = i * s.units - start - s.cost, hi = lo + s.units;
    begin = lo <= 0 ? 0 : (lo >= len ? len : (int)lo & -s.snap);
    end = hi <= 0 ? 0 : (hi >= len ? len : (int)hi & -s.snap);
}
// The pieces of a span, in order.
struct PieceCursor {
    int b, start, len, begin, end;
    __device__ __forceinline__ bool load(const StreamParams &p, const SpanPlan &s, long long span) {
        // from sequence b on, the first one with keys in the span; false behind the last
        for (; b < p.batch; ++b) {
            start = p.cu_seq_k[b];
            const long long at = axis_start(s, b, start);
            if (at >= (span + 1) * s.units) return false;
            len = sequence_keys(p, b, start);
            if (len == 0) continue;
            span_piece(s, span, at, len, begin, end);
            if (begin < end) return true;
        }
        return false;
    }
};

// Largest b in [0, batch) that begins on the axis at or before x, by the lanes of a warp together (0 if there is none).
__device__ __forceinline__ int find_sequence(const SpanPlan &s, const int *cu, int batch, long long x, int lane) {
    int lo = 0, n = batch;
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lane * step;
        const unsigned hit = __ballot_sync(0xffffffffu, at < n && axis_start(s, lo + at, cu[lo + at]) <= x);
        const int count = __popc(hit);
        const int off = count > 0 ? (count - 1) * step : 0;
        lo += off;
        n = n - off < step ? n - off : step;
    }
    return lo;
}
#endif

}  // namespace da
