// Joins what the key-stream kernel (da_stream_kernel.cuh) left in pieces, and the parts of a shared prefix:
//     o = sum_i e^(lse_i - L) o_i,   L = log sum_i e^(lse_i)
// A row is a (sequence, query head); a sequence that one CTA finished is skipped, an empty one gets zeros and -inf.
// Bound: latency (a few loads behind one another), so the kernel is launched while the stream kernel still runs, and where
// rows are few -- then they have many parts -- kWarps warps share a row's parts.
#include "da_internal.h"
#include "da_stream.h"

namespace da {
namespace {

constexpr int kMergeWarps = 8;

template <int D, int kWarps>
__global__ void __launch_bounds__(kMergeWarps * 32) da_stream_merge_kernel(const StreamMergeParams p) {
    constexpr int kVec = (D + 127) / 128;  // 16-byte groups of a lane
    constexpr int kRows = kMergeWarps / kWarps;
    __shared__ float4 acc_s[kWarps > 1 ? kMergeWarps : 1][kVec * 32];
    __shared__ float2 stat_s[kWarps > 1 ? kMergeWarps : 1];  // reference maximum and sum of each warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int slice = warp % kWarps;  // parts slice * 32 .. + 31 of every kWarps * 32
    const int head = min(blockIdx.x * kRows + warp / kWarps, p.s.head_q - 1);  // (a row may be done twice, alike)
    const int b = blockIdx.y;
    pdl_wait();
    const SpanPlan plan = span_plan(p.s);
    const int cu = p.s.cu_seq_k[b];
    const long long start = axis_start(plan, b, cu);
    int len = p.s.cu_seq_k[b + 1] - cu;
    if (len < 0) len = 0;
    const long long row = (long long)b * p.s.head_q + head;

    // stream parts: spans first_span .. first_span + spans - 1, or the whole sequence in own_o
    long long first_span = 0;
    int spans = 0;
    bool whole = false;
    if (len > 0) {
        first_span = start / plan.units;
        spans = (int)((start + plan.cost + len - 1) / plan.units - first_span) + 1;
        int begin, end;
        for (int i = 0; i < 2 && i < spans; ++i) {
            span_piece(plan, first_span + i, start, len, begin, end);
            whole |= begin == 0 && end == len;
        }
    }
    if (whole && p.s.o) return;  // the stream kernel has written it (the same for all rows of the block)
    const int prefix_parts = p.prefix_o ? prefix_parts_of(p.prefix, head / p.s.group, b) : 0;
    const int parts = prefix_parts + (whole ? 1 : spans);
    // Record of part i: where its row and its log-sum-exp are; false for a span that got none of the sequence's keys.
    auto locate = [&](int i, const float *&o, float &lse) {
        if (i < prefix_parts) {
            const long long at = (long long)i * p.s.batch * p.s.head_q + row;
            o = p.prefix_o + at * D;
            lse = p.prefix_lse[at];
        } else if (whole) {
            o = p.s.own_o + row * D;
            lse = p.s.own_lse[row];
        } else {
            const long long span = first_span + (i - prefix_parts);
            int begin, end;
            span_piece(plan, span, start, len, begin, end);
            const long long at = (span * 2 + (begin == 0 ? 1 : 0)) * p.s.head_q + head;
            o = p.s.part_o + at * D;
            lse = begin < end ? p.s.part_lse[at] : -INFINITY;
        }
    };

    float ref = -INFINITY, sum = 0.0f;
    bool odd = false;  // a part that is NaN makes the row NaN
    float4 acc[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = slice * 32; i0 < parts; i0 += kWarps * 32) {
        const float *mine = nullptr;
        float lse = -INFINITY;
        if (i0 + lane < parts) locate(i0 + lane, mine, lse);
        odd |= lse != lse;
        float top = lse;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (top > ref) {
            const float shrink = exp2f((ref - top) * kLog2e);
            ref = top;
            sum *= shrink;
#pragma unroll
            for (int v = 0; v < kVec; ++v) acc[v] = make_float4(acc[v].x * shrink, acc[v].y * shrink, acc[v].z * shrink, acc[v].w * shrink);
        }
        const float w = lse == -INFINITY ? 0.0f : exp2f((lse - ref) * kLog2e);
        sum += w;
        const int n = min(32, parts - i0);
        for (int i = 0; i < n; i += 8) {
            float4 y[8][kVec];
            float wi[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                wi[k] = __shfl_sync(0xffffffffu, w, (i + k) & 31);
                const float4 *o = reinterpret_cast<const float4 *>(__shfl_sync(0xffffffffu, (unsigned long long)mine, (i + k) & 31));
                const bool read = i + k < n && wi[k] > 0.0f;
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const int at = v * 32 + lane;
                    y[k][v] = read && at * 4 < D ? __ldcg(o + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
                if (!read) wi[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    acc[v].x = fmaf(wi[k], y[k][v].x, acc[v].x);
                    acc[v].y = fmaf(wi[k], y[k][v].y, acc[v].y);
                    acc[v].z = fmaf(wi[k], y[k][v].z, acc[v].z);
                    acc[v].w = fmaf(wi[k], y[k][v].w, acc[v].w);
                }
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (__any_sync(0xffffffffu, odd)) sum = __uint_as_float(0x7fffffffu);
    if (kWarps > 1) {
        if (lane == 0) stat_s[warp] = make_float2(ref, sum);
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc_s[warp][v * 32 + lane] = acc[v];
        __syncthreads();
        if (slice != 0) return;
        float top = ref;
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, stat_s[warp + k].x);
        sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float2 st = stat_s[warp + k];
            const float w = st.x == -INFINITY ? (st.y != st.y ? st.y : 0.0f) : exp2f((st.x - top) * kLog2e);
            sum = fmaf(w, st.y, sum);
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const float4 y = acc_s[warp + k][v * 32 + lane];
                acc[v].x = fmaf(w, y.x, acc[v].x);
                acc[v].y = fmaf(w, y.y, acc[v].y);
                acc[v].z = fmaf(w, y.z, acc[v].z);
                acc[v].w = fmaf(w, y.w, acc[v].w);
            }
        }
        ref = top;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);  // (NaN stays NaN)
    uint16_t *dst = static_cast<uint16_t *>(p.o) + (long long)b * p.s.o_row_stride + (long long)head * D;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        const int at = v * 32 + lane;
        if (at * 4 >= D) continue;
        const float y[4] = {acc[v].x * inv, acc[v].y * inv, acc[v].z * inv, acc[v].w * inv};
        ushort4 h;
        uint16_t *e = reinterpret_cast<uint16_t *>(&h);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            e[i] = p.s.q_bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y[i])) : __half_as_ushort(__float2half_rn(y[i]));
        *reinterpret_cast<ushort4 *>(dst + at * 4) = h;
    }
    if (lane == 0 && p.lse) p.lse[row] = sum > 0.0f ? ref + logf(sum) : (sum == 0.0f ? -INFINITY : sum);
}

template <int D>
cudaError_t launch_merge_dim(const StreamMergeParams &p, cudaStream_t s, bool overlap) {
    // Up to 2 048 rows, a block each: 220 rows of 75 parts take 6 us instead of 42.  Above, a warp each.
    if ((long long)p.s.batch * p.s.head_q <= 2048)
        return launch_kernel(da_stream_merge_kernel<D, 8>, dim3(p.s.head_q, p.s.batch), kMergeWarps * 32, 0, s, overlap, p);
    return launch_kernel(da_stream_merge_kernel<D, 1>, dim3((p.s.head_q + 7) / 8, p.s.batch), kMergeWarps * 32, 0, s, overlap, p);
}

}  // namespace

cudaError_t launch_stream_merge(const StreamMergeParams &p, cudaStream_t s, bool overlap) {
    count_launch();
    switch (p.dim) {
        case 64: return launch_merge_dim<64>(p, s, overlap);
        case 96: return launch_merge_dim<96>(p, s, overlap);
        case 128: return launch_merge_dim<128>(p, s, overlap);
        case 256: return launch_merge_dim<256>(p, s, overlap);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace da
