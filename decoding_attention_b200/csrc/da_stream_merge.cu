// Joins what the key-stream kernel (da_stream_kernel.cuh) left in pieces, and the parts of a shared prefix:
//     o = sum_i e^(lse_i - L) o_i,   L = log sum_i e^(lse_i)
// A row is a (sequence, query head); a sequence that one CTA finished is skipped, an empty one gets zeros and -inf.
// Bound: latency (a few loads behind one another; it ends 3 to 11 us after the stream kernel), so the kernel is launched
// while the stream kernel still runs and looks up where its parts are before it waits, and where rows are few -- then they
// have many parts -- kWarps warps share a row's parts.
#include "da_internal.h"
#include "da_stream.h"

namespace da {
namespace {

constexpr int kMergeWarps = 8;

// A row's accumulator: dims 4 lane .. 4 lane + 3 (and 128 further on) of a warp.
template <int D>
struct RowSum {
    static constexpr int kVec = (D + 127) / 128;
    float ref, sum;  // reference maximum, sum of the weights in this lane
    float4 acc[kVec];
    __device__ __forceinline__ void clear() {
        ref = -INFINITY;
        sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    __device__ __forceinline__ void scale(float f) {
        sum *= f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = make_float4(acc[v].x * f, acc[v].y * f, acc[v].z * f, acc[v].w * f);
    }
    __device__ __forceinline__ void add(float w, const float4 (&y)[kVec]) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            acc[v].x = fmaf(w, y[v].x, acc[v].x);
            acc[v].y = fmaf(w, y[v].y, acc[v].y);
            acc[v].z = fmaf(w, y[v].z, acc[v].z);
            acc[v].w = fmaf(w, y[v].w, acc[v].w);
        }
    }
};

// kWarps warps share a row; with kWarps = 1 a warp does `heads_per_warp` rows of a sequence one after another.
template <int D, int kWarps>
__global__ void __launch_bounds__(kMergeWarps * 32, kWarps == 1 ? 5 : 3) da_stream_merge_kernel(const StreamMergeParams p, const int heads_per_warp) {
    constexpr int kVec = RowSum<D>::kVec;
    constexpr int kRows = kMergeWarps / kWarps;
    constexpr int kBatch = (kWarps == 1 ? 4 : 8) / kVec;  // records in flight: fewer where rows are many, for more warps
    __shared__ float4 acc_s[kWarps > 1 ? kMergeWarps : 1][kVec * 32];
    __shared__ float2 stat_s[kWarps > 1 ? kMergeWarps : 1];  // reference maximum and sum of each warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int slice = warp % kWarps;  // this warp's parts: slice, slice + kWarps, ...
    const int b = blockIdx.y;
    // Where the parts are depends on the lengths alone, which were there before the stream kernel started.
    const SpanPlan plan = span_plan(p.s);
    const int cu = p.s.cu_seq_k[b];
    const long long start = axis_start(plan, b, cu);
    const int len = sequence_keys(p.s, b, cu);

    // stream parts: spans first_span .. first_span + spans - 1, or the whole sequence in own_o
    long long first_span = 0;
    int spans = 0;
    bool whole = false;
    if (len > 0) {
        first_span = axis_div(start, plan.units);
        spans = (int)(axis_div(start + plan.cost + len - 1, plan.units) - first_span) + 1;
        // (lengths that are not cumulative would point outside the workspace)
        if (first_span < 0 || first_span >= p.s.spans) first_span = spans = 0;
        if (first_span + spans > p.s.spans) spans = (int)(p.s.spans - first_span);
        int begin, end;
        for (int i = 0; i < 2 && i < spans; ++i) {
            span_piece(plan, first_span + i, start, len, begin, end);
            whole |= begin == 0 && end == len;
        }
    }
    if (whole && p.s.o) {  // the stream kernel has written it (the same for all rows of the block)
        pdl_wait();
        return;
    }
    PrefixGrid grid = p.prefix;
    if (p.prefix_o) grid.cta_tiles = prefix_run(grid, plan.total - (long long)p.s.batch * plan.cost);
    bool waited = false;
    for (int r = 0; r < (kWarps == 1 ? heads_per_warp : 1); ++r) {
        // (past the last head a row is done twice, alike)
        const int head = min((blockIdx.x * kRows + warp / kWarps) * (kWarps == 1 ? heads_per_warp : 1) + r, p.s.head_q - 1);
        const long long row = (long long)b * p.s.head_q + head;
        const int prefix_parts = p.prefix_o ? prefix_parts_of(grid, head / p.s.group, b) : 0;
        const int parts = prefix_parts + (whole ? 1 : spans);
        // Record of part i: its row and its log-sum-exp; NULL for a span that got none of the sequence's keys.
        auto locate = [&](int i, const float *&o, const float *&lse) {
            if (i >= parts) return;
            if (i < prefix_parts) {
                const long long at = (long long)i * p.s.batch * p.s.head_q + row;
                o = p.prefix_o + at * D;
                lse = p.prefix_lse + at;
            } else if (whole) {
                o = p.s.own_o + row * D;
                lse = p.s.own_lse + row;
            } else {
                const long long span = first_span + (i - prefix_parts);
                int begin, end;
                span_piece(plan, span, start, len, begin, end);
                const long long at = (span * 2 + (begin == 0 ? 1 : 0)) * p.s.head_q + head;
                if (begin < end) {
                    o = p.s.part_o + at * D;
                    lse = p.s.part_lse + at;
                }
            }
        };

        RowSum<D> x;
        x.clear();
        bool odd = false;  // a part that is NaN makes the row NaN
        for (int j0 = 0; j0 * kWarps + slice < parts || j0 == 0; j0 += 32) {
            const float *mine = nullptr, *mine_lse = nullptr;
            locate((j0 + lane) * kWarps + slice, mine, mine_lse);
            const int n = min(32, (parts - slice + kWarps - 1) / kWarps - j0);
            if (!waited) pdl_wait();
            waited = true;
            const float lse = mine_lse ? __ldcg(mine_lse) : -INFINITY;
            float w = 0.0f;
            for (int i = 0; i < n; i += kBatch) {
                float4 y[kBatch][kVec];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const float4 *o = reinterpret_cast<const float4 *>(__shfl_sync(0xffffffffu, (unsigned long long)mine, (i + k) & 31));
#pragma unroll
                    for (int v = 0; v < kVec; ++v) {
                        const int at = v * 32 + lane;
                        y[k][v] = o && i + k < n && at * 4 < D ? __ldcg(o + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
                if (i == 0) {  // (the first records are on their way while the weights are worked out)
                    odd |= lse != lse;
                    float top = lse;
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    if (top > x.ref) {
                        x.scale(exp2f((x.ref - top) * kLog2e));
                        x.ref = top;
                    }
                    w = lse == -INFINITY ? 0.0f : exp2f((lse - x.ref) * kLog2e);
                    x.sum += w;
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const float wi = __shfl_sync(0xffffffffu, w, (i + k) & 31);
                    if (i + k < n && wi != 0.0f) x.add(wi, y[k]);  // (a part without keys has no row)
                }
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x.sum += __shfl_xor_sync(0xffffffffu, x.sum, d);
        if (__any_sync(0xffffffffu, odd)) x.sum = __uint_as_float(0x7fffffffu);
        if (kWarps > 1) {
            if (lane == 0) stat_s[warp] = make_float2(x.ref, x.sum);
#pragma unroll
            for (int v = 0; v < kVec; ++v) acc_s[warp][v * 32 + lane] = x.acc[v];
            __syncthreads();
            if (slice != 0) return;
            float top = x.ref;
#pragma unroll
            for (int k = 1; k < kWarps; ++k) top = fmaxf(top, stat_s[warp + k].x);
            x.clear();
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float2 st = stat_s[warp + k];
                const float w = st.x == -INFINITY ? (st.y != st.y ? st.y : 0.0f) : exp2f((st.x - top) * kLog2e);
                x.sum = fmaf(w, st.y, x.sum);
                float4 y[kVec];
#pragma unroll
                for (int v = 0; v < kVec; ++v) y[v] = acc_s[warp + k][v * 32 + lane];
                x.add(w, y);
            }
            x.ref = top;
        }
        const float inv = x.sum > 0.0f ? 1.0f / x.sum : (x.sum == 0.0f ? 0.0f : x.sum);  // (NaN stays NaN)
        uint16_t *dst = static_cast<uint16_t *>(p.o) + (long long)b * p.s.o_row_stride + (long long)head * D;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const int at = v * 32 + lane;
            if (at * 4 >= D) continue;
            const float y[4] = {x.acc[v].x * inv, x.acc[v].y * inv, x.acc[v].z * inv, x.acc[v].w * inv};
            ushort4 h;
            uint16_t *e = reinterpret_cast<uint16_t *>(&h);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                e[i] = p.s.q_bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y[i])) : __half_as_ushort(__float2half_rn(y[i]));
            *reinterpret_cast<ushort4 *>(dst + at * 4) = h;
        }
        if (lane == 0 && p.lse) p.lse[row] = x.sum > 0.0f ? x.ref + logf(x.sum) : (x.sum == 0.0f ? -INFINITY : x.sum);
    }
    // The next call's kernel may start now, and not earlier: its big blocks, put down between the small ones of this kernel,
    // would find the register file in pieces, and some SMs then hold one block less until their first ones end (256
    // sequences of 512-4096 FP8 keys, calls back to back: 265 us where 212 are enough).
    pdl_launch_dependents();
}

template <int D, int kWarps>
cudaError_t launch_merge_warps(const StreamMergeParams &p, int heads_per_warp, cudaStream_t s) {
    const int heads = kMergeWarps / kWarps * heads_per_warp;
    return launch_kernel(da_stream_merge_kernel<D, kWarps>, dim3((p.s.head_q + heads - 1) / heads, p.s.batch), kMergeWarps * 32, 0, s,
                         true, p, heads_per_warp);
}
template <int D>
cudaError_t launch_merge_dim(const StreamMergeParams &p, cudaStream_t s) {
    // Parts of a row, as far as the host can tell: those of the prefix and the sequence's share of the spans.  A warp for
    // every four of them, if the blocks then still fit the SMs at once (three each; twice that for two warps and many parts).
    // Otherwise a warp a row, and above five blocks an SM two rows a warp, which share the search for their parts.
    const int parts = (p.prefix_o ? p.prefix.max_parts : 0) + 1 + p.s.spans / p.s.batch;
    auto blocks = [&](int warps) { return (long long)p.s.batch * ((p.s.head_q * warps + 7) / 8); };
    const int at_once = 3 * p.sms;
    if (parts > 16 && blocks(8) <= at_once) return launch_merge_warps<D, 8>(p, 1, s);
    if (parts > 8 && blocks(4) <= at_once) return launch_merge_warps<D, 4>(p, 1, s);
    if (parts > 4 && blocks(2) <= (parts > 8 ? 2 * at_once : at_once)) return launch_merge_warps<D, 2>(p, 1, s);
    const bool many = blocks(1) > 5 * p.sms && p.s.head_q > 8;
    return launch_merge_warps<D, 1>(p, many ? 2 : 1, s);
}

}  // namespace

cudaError_t launch_stream_merge(const StreamMergeParams &p, cudaStream_t s) {
    count_launch();
    switch (p.dim) {
        case 64: return launch_merge_dim<64>(p, s);
        case 96: return launch_merge_dim<96>(p, s);
        case 128: return launch_merge_dim<128>(p, s);
        case 256: return launch_merge_dim<256>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace da
