// Joins what the key-stream kernel (da_stream_kernel.cuh) left in pieces, and the parts of a shared prefix:
//     o = sum_i e^(lse_i - L) o_i,   L = log sum_i e^(lse_i)
// One warp per (sequence, query head); a sequence that one CTA finished is skipped, an empty one gets zeros and -inf.
// Bound: latency (a few loads behind one another); the kernel is launched while the stream kernel still runs.
#include "da_internal.h"
#include "da_stream.h"

namespace da {
namespace {

constexpr int kMergeWarps = 8;

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) da_stream_merge_kernel(const StreamMergeParams p) {
    constexpr int kVec = (D + 127) / 128;  // 16-byte groups of a lane
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.x * kMergeWarps + threadIdx.x / 32;
    const int b = blockIdx.y;
    pdl_wait();
    if (head >= p.s.head_q) return;
    const SpanPlan plan = span_plan(p.s);
    const int start = p.s.cu_seq_k[b];
    int len = p.s.cu_seq_k[b + 1] - start;
    if (len < 0) len = 0;
    const long long row = (long long)b * p.s.head_q + head;

    // stream parts: span first_span + i for i in [0, spans), or the whole sequence in own_o
    long long first_span = 0;
    int spans = 0;
    bool whole = false;
    if (len > 0) {
        first_span = (start - plan.first) / plan.keys;
        spans = (int)((start + (long long)len - 1 - plan.first) / plan.keys - first_span) + 1;
        int begin, end;
        for (int i = 0; i < 2 && i < spans; ++i) {
            span_piece(plan, first_span + i, start, len, begin, end);
            whole |= begin == 0 && end == len;
        }
    }
    if (whole && p.s.o) return;  // the stream kernel has written it
    const int stream_parts = whole ? 1 : spans;
    const int prefix_parts = p.prefix_o ? prefix_parts_of(p.prefix, head / p.s.group, b) : 0;
    const int parts = prefix_parts + stream_parts;
    auto part_lse = [&](int i) -> float {
        if (i < prefix_parts) return p.prefix_lse[(long long)i * p.s.batch * p.s.head_q + row];
        if (whole) return p.s.own_lse[row];
        i -= prefix_parts;
        int begin, end;
        span_piece(plan, first_span + i, start, len, begin, end);
        if (begin >= end) return -INFINITY;
        return p.s.part_lse[((first_span + i) * 2 + (begin == 0 ? 1 : 0)) * p.s.head_q + head];
    };
    auto part_o = [&](int i) -> const float * {
        if (i < prefix_parts) return p.prefix_o + ((long long)i * p.s.batch * p.s.head_q + row) * D;
        if (whole) return p.s.own_o + row * D;
        i -= prefix_parts;
        int begin, end;
        span_piece(plan, first_span + i, start, len, begin, end);
        return p.s.part_o + (((first_span + i) * 2 + (begin == 0 ? 1 : 0)) * p.s.head_q + head) * D;
    };

    float top = -INFINITY;
    bool odd = false;  // a part that is NaN makes the row NaN
    for (int i = lane; i < parts; i += 32) {
        const float x = part_lse(i);
        odd |= x != x;
        top = fmaxf(top, x);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    odd = __any_sync(0xffffffffu, odd);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < parts; i0 += 32) {
        const float x = i0 + lane < parts ? part_lse(i0 + lane) : -INFINITY;
        const float w = exp2f((x - ref) * kLog2e);
        sum += w;
        const int n = min(32, parts - i0);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            if (!(wi != 0.0f)) continue;  // (also a piece that was never written)
            const float4 *o = reinterpret_cast<const float4 *>(part_o(i0 + i));
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const int at = v * 32 + lane;
                if (at * 4 < D) {
                    const float4 y = __ldcg(o + at);
                    acc[v].x = fmaf(wi, y.x, acc[v].x);
                    acc[v].y = fmaf(wi, y.y, acc[v].y);
                    acc[v].z = fmaf(wi, y.z, acc[v].z);
                    acc[v].w = fmaf(wi, y.w, acc[v].w);
                }
            }
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    if (odd || sum != sum) inv = __uint_as_float(0x7fffffffu);
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
    if (lane == 0 && p.lse) p.lse[row] = odd ? __uint_as_float(0x7fffffffu) : (sum > 0.0f ? ref + logf(sum) : (sum == 0.0f ? -INFINITY : sum));
}

}  // namespace

cudaError_t launch_stream_merge(const StreamMergeParams &p, cudaStream_t s, bool overlap) {
    const dim3 grid((p.s.head_q + kMergeWarps - 1) / kMergeWarps, p.s.batch);
    count_launch();
    switch (p.dim) {
        case 64: return launch_kernel(da_stream_merge_kernel<64>, grid, kMergeWarps * 32, 0, s, overlap, p);
        case 96: return launch_kernel(da_stream_merge_kernel<96>, grid, kMergeWarps * 32, 0, s, overlap, p);
        case 128: return launch_kernel(da_stream_merge_kernel<128>, grid, kMergeWarps * 32, 0, s, overlap, p);
        case 256: return launch_kernel(da_stream_merge_kernel<256>, grid, kMergeWarps * 32, 0, s, overlap, p);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace da
