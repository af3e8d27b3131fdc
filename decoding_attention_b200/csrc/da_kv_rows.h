// Launch parameters of the row kernels of a quantised KV cache (da_kv_rows.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace da {

// Division of 31-bit numbers by a constant: (umulhi(n, mul) + n) >> shift (Granlund and Montgomery).
struct FastDiv {
    uint32_t mul;
    int shift;
};
inline FastDiv make_fast_div(uint32_t d) {
    int s = 0;
    while ((1ull << s) < d) ++s;
    return {(uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

struct KvRowsParams {
    void *k, *v;              // rows [tokens, head_k, dim]: read by the writer, written by the reader
    void *k_cache, *v_cache;  // codes [cache_rows, head_k, dim]
    float *k_scale, *v_scale; // [cache_rows, head_k]
    const int64_t *slots;     // cache row of each token, or NULL: token i and row i
    long long k_row_stride, v_row_stride;  // elements between tokens of k / v
    long long cache_rows;
    uint32_t rows;  // tokens * head_k
    int head_k;
    FastDiv by_heads;
};
// x_dtype: type of k and v (0 fp16, 1 bf16, 2 fp32, reading only); kvq: 1 FP8 e4m3, 2 int8, 3 int4.
cudaError_t launch_kv_rows(const KvRowsParams &p, int dim, int x_dtype, int kvq, bool write, cudaStream_t s);

}  // namespace da
