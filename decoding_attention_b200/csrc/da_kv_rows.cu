// Rows of a quantised KV cache: writing them from 16-bit rows and reading them back.
//
// A row x is one token and one KV head, D values.  With Q the largest code of the format (448 for FP8 e4m3, 127
// for int8, 7 for int4) and a = max |x|:
//     scale = fl32(a / Q),   code = rn(x * fl32(Q / a)),   x is read back as rn(code * scale).
// The product is rounded ONCE, from its exact value: for integers by an fma that adds 1.5 * 2^23 (whose ulp is 1),
// for e4m3 by truncating to 24 bits with a sticky last bit before the hardware conversion -- so the codes are a
// function of the definition and not of an order of operations.  Rows with a < 2^-100 become zeros with scale 0
// (both quotients stay normal numbers); a row that holds an infinity or a NaN gets scale NaN and codes 0, so that
// whatever reads it sees NaN.
//
// Bound: HBM.  A row costs 2D bytes on the 16-bit side and D (or D / 2) + 4 on the other; nothing is read twice.  32 768
// tokens x 8 KV heads of 128 into int8: 32 us, the copy rate; 131 072 tokens out of FP8: 125 us, the copy rate.  Single
// tokens: 1.3 us of a stream's time, a launch.
// A row belongs to L = D / 16 lanes that hold two pieces of 8 values (16-byte accesses on the 16-bit side, lanes side by
// side); a thread has kRows rows in flight, since the slot, the row and (reading) the scale are a chain of two loads.
// Writing is close to the issue limit, so what is done once a row is done for kRows rows at a time: the maxima of four
// rows are joined by reduce-scatter (four shuffles for L = 8 where four xor reductions take twelve), after which every lane
// has the maximum of one row, and the two quotients are worked out once for all of them (a shuffle a row hands them back).
#include "da_internal.h"
#include "da_kv_rows.h"

namespace da {
namespace {

constexpr int kThreads = 256;

// Lanes of a row and 8-value chunks of a lane.
template <int D>
struct RowCfg {
    static constexpr int kLanes = D == 96 ? 4 : D / 16;
    static constexpr int kChunks = D / 8 / kLanes;
};

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv &d) { return (__umulhi(n, d.mul) + n) >> d.shift; }

template <int KVQ>
__device__ __forceinline__ constexpr float code_max() {
    return KVQ == 1 ? 448.0f : (KVQ == 2 ? 127.0f : 7.0f);
}

// x * inv rounded once to an integer; the low bits of the result are the code in two's complement.
__device__ __forceinline__ uint32_t round_code(float x, float inv) {
    return __float_as_uint(__fmaf_rn(x, inv, 12582912.0f));
}
// x * inv cut to 24 bits, with the last bit set when something was cut off: a second rounding to fewer bits then
// gives what one rounding of the exact product would.
__device__ __forceinline__ float product_sticky(float x, float inv) {
    const float p = __fmul_rz(x, inv);
    const float rest = __fmaf_rn(x, inv, -p);
    return __uint_as_float(__float_as_uint(p) | (rest != 0.0f ? 1u : 0u));
}

template <int KVQ>
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&x)[8], float inv) {
    if (KVQ == 1) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 a = {product_sticky(x[4 * i], inv), product_sticky(x[4 * i + 1], inv)};
            const float2 b = {product_sticky(x[4 * i + 2], inv), product_sticky(x[4 * i + 3], inv)};
            w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                   ((uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16);
        }
        *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    } else if (KVQ == 2) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t lo = __byte_perm(round_code(x[4 * i], inv), round_code(x[4 * i + 1], inv), 0x0040);
            const uint32_t hi = __byte_perm(round_code(x[4 * i + 2], inv), round_code(x[4 * i + 3], inv), 0x0040);
            w[i] = __byte_perm(lo, hi, 0x5410);
        }
        *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= (round_code(x[i], inv) & 15u) << (4 * i);
        *reinterpret_cast<uint32_t *>(dst) = w;
    }
}

// The larger 16-bit magnitude of each half, sign bits cleared: magnitudes compare as integers, and infinities and NaN come
// out above every number.
__device__ __forceinline__ uint32_t max_magnitude(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <typename T>
__device__ __forceinline__ float magnitude(uint32_t bits);
template <>
__device__ __forceinline__ float magnitude<__half>(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
}
template <>
__device__ __forceinline__ float magnitude<__nv_bfloat16>(uint32_t bits) {
    return __uint_as_float(bits << 16);
}

// blockIdx.y: 0 the K rows, 1 the V rows.  Row r = token * head_k + head.
template <typename T, int D, int KVQ, int kRows>
__global__ void __launch_bounds__(kThreads) da_kv_write_kernel(const KvRowsParams p) {
    using C = RowCfg<D>;
    constexpr int L = C::kLanes;
    constexpr int kRowBytes = KVQ == 3 ? D / 2 : D;
    constexpr int kBlockRows = kThreads / L;
    static_assert(kRows == 1 || kRows == 4, "rows of a thread");
    const T *__restrict__ src = static_cast<const T *>(blockIdx.y ? p.v : p.k);
    const long long src_stride = blockIdx.y ? p.v_row_stride : p.k_row_stride;
    uint8_t *__restrict__ cache = static_cast<uint8_t *>(blockIdx.y ? p.v_cache : p.k_cache);
    float *__restrict__ scales = blockIdx.y ? p.v_scale : p.k_scale;
    pdl_wait();  // the kernel before this one may still be running
    const int lane = threadIdx.x % L;
    const uint32_t first = blockIdx.x * (uint32_t)(kBlockRows * kRows) + threadIdx.x / L;

    uint4 raw[kRows][C::kChunks];
    long long dst[kRows];  // row of the cache, or -1
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = first + i * kBlockRows;
        dst[i] = -1;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) raw[i][c] = make_uint4(0, 0, 0, 0);
        if (r < p.rows) {
            const uint32_t token = fast_div(r, p.by_heads), head = r - token * (uint32_t)p.head_k;
            const long long slot = p.slots ? p.slots[token] : (long long)token;
            const T *row = src + (long long)token * src_stride + (long long)head * D;
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) raw[i][c] = __ldcs(reinterpret_cast<const uint4 *>(row) + lane + c * L);
            if (slot >= 0 && slot < p.cache_rows) dst[i] = slot * p.head_k + head;
        }
    }
    uint32_t top[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        uint32_t t = 0;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
            const uint4 &x = raw[i][c];
            const uint32_t m = 0x7fff7fffu;
            t = max_magnitude(t, max_magnitude(max_magnitude(x.x & m, x.y & m), max_magnitude(x.z & m, x.w & m)));
        }
        top[i] = t;
    }
    // Lane q of a row's lanes comes to hold row `mine` = the top two bits of q (all rows of the one there is).
    uint32_t t = top[0];
    int mine = 0;
    if (kRows == 4) {
        const bool up = lane & (L / 2), up2 = lane & (L / 4);
        const uint32_t give0 = up ? top[0] : top[2 % kRows], give1 = up ? top[1 % kRows] : top[3 % kRows];
        const uint32_t keep0 = up ? top[2 % kRows] : top[0], keep1 = up ? top[3 % kRows] : top[1 % kRows];
        const uint32_t a = max_magnitude(keep0, __shfl_xor_sync(0xffffffffu, give0, L / 2));
        const uint32_t b = max_magnitude(keep1, __shfl_xor_sync(0xffffffffu, give1, L / 2));
        t = max_magnitude(up2 ? b : a, __shfl_xor_sync(0xffffffffu, up2 ? a : b, L / 4));
        mine = (up ? 2 : 0) + (up2 ? 1 : 0);
#pragma unroll
        for (int d = L / 8; d > 0; d >>= 1) t = max_magnitude(t, __shfl_xor_sync(0xffffffffu, t, d));
    } else {
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) t = max_magnitude(t, __shfl_xor_sync(0xffffffffu, t, d));
    }
    const float amax = magnitude<T>(max(t & 0xffffu, t >> 16));
    float scale = 0.0f, inv = 0.0f;
    if (!(amax <= 3.4028235e38f)) {  // an infinity or a NaN
        scale = inv = __uint_as_float(0x7fffffffu);
    } else if (amax >= 7.8886091e-31f) {  // 2^-100
        scale = __fdiv_rn(amax, code_max<KVQ>());
        inv = __fdiv_rn(code_max<KVQ>(), amax);
    }
    long long own = dst[0];
#pragma unroll
    for (int i = 1; i < kRows; ++i) own = mine == i ? dst[i] : own;
    if (own >= 0 && (lane & (kRows == 4 ? L / 4 - 1 : L - 1)) == 0) scales[own] = scale;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        float f = __shfl_sync(0xffffffffu, inv, kRows == 4 ? i * (L / 4) : 0, L);
        const bool odd = f != f;
        if (dst[i] < 0) continue;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
            if (odd) raw[i][c] = make_uint4(0, 0, 0, 0);
            float x[8];
            unpack8<T>(raw[i][c], x);
            store_codes<KVQ>(cache + dst[i] * kRowBytes + (lane + c * L) * (KVQ == 3 ? 4 : 8), x, odd ? 0.0f : f);
        }
    }
    pdl_launch_dependents();  // (at the end: see da_stream_merge.cu)
}

template <typename T>
__device__ __forceinline__ void store8(T *dst, const float (&x)[8]) {
    uint4 w;
    T *h = reinterpret_cast<T *>(&w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = from_float<T>(x[e]);
    __stcs(reinterpret_cast<uint4 *>(dst), w);
}
template <>
__device__ __forceinline__ void store8<float>(float *dst, const float (&x)[8]) {
    __stcs(reinterpret_cast<float4 *>(dst), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4 *>(dst) + 1, make_float4(x[4], x[5], x[6], x[7]));
}

template <typename T, int D, int KVQ, int kRows>
__global__ void __launch_bounds__(kThreads) da_kv_read_kernel(const KvRowsParams p) {
    using C = RowCfg<D>;
    constexpr int kRowBytes = KVQ == 3 ? D / 2 : D;
    constexpr int kBlockRows = kThreads / C::kLanes;
    T *__restrict__ dst = static_cast<T *>(blockIdx.y ? p.v : p.k);
    const long long dst_stride = blockIdx.y ? p.v_row_stride : p.k_row_stride;
    const uint8_t *__restrict__ cache = static_cast<const uint8_t *>(blockIdx.y ? p.v_cache : p.k_cache);
    const float *__restrict__ scales = blockIdx.y ? p.v_scale : p.k_scale;
    pdl_wait();
    const int lane = threadIdx.x % C::kLanes;
    const uint32_t total = p.rows;
    const uint32_t first = blockIdx.x * (uint32_t)(kBlockRows * kRows) + threadIdx.x / C::kLanes;

    uint2 raw[kRows][C::kChunks];
    float scale[kRows];
    long long slot[kRows];
    uint32_t token[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = first + i * kBlockRows;
        token[i] = fast_div(r < total ? r : 0, p.by_heads);
        slot[i] = r < total ? (p.slots ? p.slots[token[i]] : (long long)token[i]) : -1;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        scale[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) raw[i][c] = make_uint2(0, 0);
        if (slot[i] < 0 || slot[i] >= p.cache_rows) continue;
        const uint32_t r = first + i * kBlockRows;
        const long long row = slot[i] * p.head_k + (r - token[i] * (uint32_t)p.head_k);
        scale[i] = scales[row];
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
            const uint8_t *q = cache + row * kRowBytes + (lane + c * C::kLanes) * (KVQ == 3 ? 4 : 8);
            if (KVQ == 3) raw[i][c].x = __ldcs(reinterpret_cast<const uint32_t *>(q));
            else raw[i][c] = __ldcs(reinterpret_cast<const uint2 *>(q));
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = first + i * kBlockRows;
        if (r >= total) continue;
        T *row = dst + (long long)token[i] * dst_stride + (long long)(r - token[i] * (uint32_t)p.head_k) * D;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
            float x[8];
            load_chunk8<__half, KVQ>(reinterpret_cast<const uint8_t *>(&raw[i][c]), x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], scale[i]);
            store8<T>(row + (lane + c * C::kLanes) * 8, x);
        }
    }
    pdl_launch_dependents();
}

// Rows of a thread.  Few rows, fewer than four blocks an SM: one each, to spread them.  (The SMs of a B200: asking the
// runtime which device is current and how many it has took 0.4 us of a call of 3.5.)
constexpr uint32_t kSms = 148;
template <typename T, int D, int KVQ>
cudaError_t launch_rows(const KvRowsParams &p, bool write, cudaStream_t s) {
    constexpr uint32_t kBlockRows = kThreads / RowCfg<D>::kLanes;
    const bool many = p.rows > 4u * kBlockRows * kSms;
    const uint32_t per_block = kBlockRows * (many ? 4u : 1u);
    const dim3 grid((p.rows + per_block - 1) / per_block, 2);
    count_launch();
    if (write) {
        if constexpr (!std::is_same<T, float>::value) {
            return many ? launch_kernel(da_kv_write_kernel<T, D, KVQ, 4>, grid, kThreads, 0, s, true, p)
                        : launch_kernel(da_kv_write_kernel<T, D, KVQ, 1>, grid, kThreads, 0, s, true, p);
        }
        return cudaErrorInvalidValue;
    }
    return many ? launch_kernel(da_kv_read_kernel<T, D, KVQ, 4>, grid, kThreads, 0, s, true, p)
                : launch_kernel(da_kv_read_kernel<T, D, KVQ, 1>, grid, kThreads, 0, s, true, p);
}

template <typename T, int D>
cudaError_t launch_kind(const KvRowsParams &p, int kvq, bool write, cudaStream_t s) {
    if (kvq == 1) return launch_rows<T, D, 1>(p, write, s);
    if (kvq == 2) return launch_rows<T, D, 2>(p, write, s);
    return launch_rows<T, D, 3>(p, write, s);
}

template <typename T>
cudaError_t launch_dim(const KvRowsParams &p, int dim, int kvq, bool write, cudaStream_t s) {
    switch (dim) {
        case 64: return launch_kind<T, 64>(p, kvq, write, s);
        case 96: return launch_kind<T, 96>(p, kvq, write, s);
        case 128: return launch_kind<T, 128>(p, kvq, write, s);
        case 256: return launch_kind<T, 256>(p, kvq, write, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_kv_rows(const KvRowsParams &p, int dim, int x_dtype, int kvq, bool write, cudaStream_t s) {
    if (x_dtype == 0) return launch_dim<__half>(p, dim, kvq, write, s);
    if (x_dtype == 1) return launch_dim<__nv_bfloat16>(p, dim, kvq, write, s);
    return launch_dim<float>(p, dim, kvq, write, s);
}

}  // namespace da
