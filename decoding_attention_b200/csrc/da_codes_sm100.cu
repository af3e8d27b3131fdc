// Decode attention over a cache of 8-bit codes on the sm_100a tensor cores, for head dims 96 and 128 and groups of at most
// four query heads: the codes are operands as they lie, nothing is widened on the way.
//
//     s_j = c ks_j (q . kc_j) [+ slope (j - (len - 1))],   o = sum_j softmax(s)_j vs_j vc_j
//
// Bound: HBM.  da_stream_kernel.cuh widens every code to fp16 in registers, which holds int8 caches to 0.72 of the HBM rate.
// Here the work of the CUDA cores is per KEY and head, not per element:
//     S^T[128 keys x N] = K[128 x D] . Qp^T,     O^T[D x N] += V^T[D x 128 keys] . Pp^T
// K and V (e4m3, or s8) are the A operands of tcgen05.mma, the other side is 8 bits wide too and comes in PIECES, columns of
// their own: q as three parts and the weights w_j = p_j vs_j as four that add up to
//   int8:  23-bit (q, signed) and 31-bit (w) fixed point, eight bits a digit; kind::i8 sums them exactly in int32
//   e4m3:  e4m3 numbers, each the rounding of what the ones before it left over, times 16 (kind::f8f6f4)
// so that q is exact to 2^-22 of its head's largest element and a weight to 2^-31 of the largest one (int8), or to 2^-11 of
// itself and 2^-29 of the largest one (e4m3).  (With three parts of a weight, 2^-23 and 2^-25, the many small weights next to a
// key that leads by 16 nats were lost from o while the denominator had them.)
//
// A CTA takes one KV head and an equal span of the batch's keys (StreamParams), three CTAs an SM.  Warps: four softmax
// warps, a thread per key of a tile (the sum over a row's keys needs no order among threads until the end), one producer
// (TMA), one issuer per contraction.  A tile is a chain -- scores, weights, the other contraction -- of about 2 us, which is
// why one or two CTAs an SM are not enough (256 x 512-4096 FP8 keys, 8 KV heads: 250 us with two, 209 with three; 131 072
// int8 keys x 32 heads: 213 and 186 us, 0.91 of the measured copy rate).  Reference maxima are common to the CTA and move
// rarely: a tile asks once (one barrier with a vote) whether a score or a weight has outgrown its reference by a factor of
// 2; if so, what the tensor core has accumulated moves to fp32 registers (a thread per dim), where it is rescaled.
//
// Tried and left out: larger groups (eight heads a CTA, two CTAs an SM: slower than the other kernel), and int4 caches
// unpacked to bytes by warps of their own (half the bytes a tile, but the same chain: 40 us where the other kernel takes 30).
#include <cfloat>

#include "da_internal.h"
#include "da_stream.h"
#include "da_tcgen05.cuh"

namespace da {
namespace {

constexpr int kKeys = 128;              // of a tile
constexpr int kRowBytes = 128;          // of a staged row: D codes, or 96 and zeros
constexpr int kTileBytes = kKeys * kRowBytes;
constexpr int kHeads = 4;
constexpr int kN = 16;                  // columns: piece * kHeads + head; of the scores' last four nobody reads
constexpr int kCtas = 3;                // per SM
constexpr int kSoftmaxThreads = 128;
constexpr int kThreads = 256;           // (the last warp only fills up)
constexpr float kHeadroom = 1.0f;       // log2 of what a score or weight may exceed its reference by
// log2 of how far the weights' reference may lie below the scores': the leading keys' V scales may be zero, and 2^(m - mw)
// has to stay a number.  Weights 2^-120 of a probability of one are far below what o can show.
constexpr float kWeightReach = 120.0f;
constexpr int kFlushTiles = 256;        // 32 768 keys: int32 holds 66 311 of 127 * 255
// Tiles of K and V, in turn.  Even, so that a slot is K's or V's for good: with an odd number the K issuer, which may be
// three tiles ahead of the other, could wait for a phase of a slot whose previous phase (a V tile) is still under way --
// and a parity wait two phases ahead passes at once.
constexpr int kSlots = 4;
static_assert(kSlots % 2 == 0, "K and V keep their slots");
constexpr int kOffQ = kSlots * kTileBytes;
constexpr int kOffP = kOffQ + kN * kRowBytes;            // two buffers
constexpr int kOffHead = kOffP + 2 * kN * kRowBytes;     // HeadState[kHeads]
constexpr int kOffRed = kOffHead + kHeads * 32;          // float2[4 warps][kHeads]
constexpr int kOffBar = kOffRed + 4 * kHeads * 8;
// slot_full / slot_empty, s_full, s_empty, p_full, p_empty [2 each], q_full
constexpr int kNumBars = 2 * kSlots + 9;
constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 32;
constexpr int kColO = 2 * kN;
constexpr int kTmemCols = 64;
static_assert(kSmemBytes + 1024 <= 228 * 1024 / kCtas, "shared memory budget");
static_assert(kOffQ % 1024 == 0 && kOffP % 1024 == 0 && (kN * kRowBytes) % 1024 == 0, "swizzle atoms");

struct HeadState {
    float factor;     // of a score: softmax scale * log2(e), q's unit
    float slope;      // ALiBi
    float m, mw;      // reference maxima of the scores and of the weights, log2
    float g;          // 2^((m - mw) / 2): one half goes to the probability, one to the V scale, so that both stay inside fp32
    float pad[3];
};

template <bool kInt>
__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
    if (kInt)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader));
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader));
}
// Instruction descriptor: D int32 or fp32, A and B s8 / u8 or e4m3, A read MN-major or K-major.
template <bool kInt>
__device__ __forceinline__ constexpr uint32_t idesc8(uint32_t b_signed, uint32_t a_mn_major, uint32_t n) {
    return ((kInt ? 2u : 1u) << 4) | ((kInt ? 1u : 0u) << 7) | ((kInt ? b_signed : 0u) << 10) | (a_mn_major << 15) | ((n >> 3) << 17) |
           ((128u >> 4) << 24);
}
// 2^e, -126 <= e <= 127
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// Whether any thread of the softmax warps says yes.
__device__ __forceinline__ bool vote_any(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x)
        : "memory");
    return r != 0;
}
// Byte of column k (a key, or a code's place) of row n in a 128-byte-swizzled operand of 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(uint32_t n, uint32_t k) { return n * 128 + (((k >> 4) ^ (n & 7)) << 4) + (k & 15); }

__device__ __forceinline__ float int_to_float(uint32_t x) {  // |x| < 2^22
    return __uint_as_float(x + 0x4b400000u) - 12582912.0f;
}
__device__ __forceinline__ uint32_t e4m3x2(__half2 x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t *>(&x)));
    return r;
}
__device__ __forceinline__ __half2 from_e4m3x2(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(x));
    return *reinterpret_cast<const __half2 *>(&r);
}

// The pieces of a span, and their tiles in the order in which all roles take them.
struct SpanWalk : PieceCursor {
    __device__ __forceinline__ int tiles() const { return (end - begin + kKeys - 1) / kKeys; }
    // ALiBi: back to front, the first tiles set the reference maxima
    __device__ __forceinline__ int key(const StreamParams &p, int i) const { return begin + (p.is_alibi ? tiles() - 1 - i : i) * kKeys; }
};

// kInt: int8 codes, else e4m3.
template <bool kInt>
__global__ void __launch_bounds__(kThreads, kCtas)
da_codes_kernel(const StreamParams p, const int dim, int *status, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kOffBar);
    uint64_t *slot_full = bars, *slot_empty = bars + kSlots;
    uint64_t *s_full = slot_empty + kSlots, *s_empty = s_full + 2, *p_full = s_empty + 2, *p_empty = p_full + 2;
    uint64_t *q_full = p_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kNumBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *fresh = abort_flag + 1;  // [2]: the tile's contraction starts the accumulator anew

    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&slot_full[i], 1);
            mbar_init(&slot_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], kSoftmaxThreads);
            mbar_init(&p_full[i], kSoftmaxThreads);
            mbar_init(&p_empty[i], 1);
        }
        mbar_init(q_full, kSoftmaxThreads);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 5) tmem_alloc(tmem_slot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (!p.chained) pdl_wait();  // the kernel before this call's may still be running
    pdl_launch_dependents();

    const SpanPlan plan = span_plan(p);
    const long long span = blockIdx.y;
    const int head_k = blockIdx.x, head0 = head_k * p.group, heads = p.group;
    bool ok = true;
    SpanWalk x;
    x.b = 0;
    bool more = span * plan.units < plan.total;
    if (more) {
        x.b = find_sequence(plan, p.cu_seq_k, p.batch, span * plan.units, lane);
        more = x.load(p, plan, span);
    }

    if (warp == 4) {
        // ---------------- TMA producer ----------------
        const int run = p.block_table && (1 << p.page_shift) < kKeys ? 1 << p.page_shift : kKeys;
        int fill = 0;
        for (; more && ok; ++x.b, more = x.load(p, plan, span)) {
            for (int i = 0; i < x.tiles() && ok; ++i) {
                const int key0 = x.key(p, i);
                // Row of every run of consecutive keys, one a lane.  A run that no page holds is fetched from row -128, i.e. as
                // zeros (its keys are masked); runs behind the end are not looked up.
                int row = -kKeys;
                const int key = key0 + lane * run;
                if (lane * run < kKeys && key < x.end) {
                    if (p.block_table) {
                        const int block = key >> p.page_shift;
                        const int page = block < p.table_blocks ? p.block_table[(long long)x.b * p.table_stride + block] : -1;
                        const long long at = ((long long)page << p.page_shift) + (key & ((1 << p.page_shift) - 1));
                        if (page >= 0 && at < p.rows) row = (int)at;
                    } else if ((long long)x.start + key < p.rows && x.start + key >= 0) {
                        row = x.start + key;
                    }
                }
                for (int kv = 0; kv < 2 && ok; ++kv, ++fill) {
                    const int st = fill % kSlots;
                    if (fill >= kSlots) ok = mbar_wait(&slot_empty[st], ((uint32_t)(fill / kSlots) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&slot_full[st], kTileBytes);
                    __syncwarp();
                    if (lane * run < kKeys)
                        tma_load_tile_3d(smem + st * kTileBytes + lane * run * kRowBytes, kv ? &tm_v : &tm_k, 0, head_k, row, &slot_full[st]);
                    __syncwarp();
                }
            }
        }
    } else if (warp == 5) {
        // ---------------- issuer of S^T = K . Qp^T ----------------
        const uint32_t leader = elect_one();
        const uint64_t k_desc = smem_desc(smem_u32(smem), 16, 1024, 2), q_desc = smem_desc(smem_u32(smem + kOffQ), 16, 1024, 2);
        constexpr uint32_t kIdesc = idesc8<kInt>(1, 0, kN);
        int t = 0, pieces = 0;
        for (; more && ok; ++x.b, more = x.load(p, plan, span), ++pieces) {
            const int n = x.tiles();
            ok = mbar_wait(q_full, (uint32_t)pieces & 1u, abort_flag);
            for (int i = 0; i < n && ok; ++i, ++t) {
                const int fill = 2 * t, st = fill % kSlots, sb = t & 1;
                ok = mbar_wait(&slot_full[st], (uint32_t)(fill / kSlots) & 1u, abort_flag);
                if (ok && t >= 2) ok = mbar_wait(&s_empty[sb], ((uint32_t)(t >> 1) & 1u) ^ 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma8<kInt>(tmem + sb * kN, k_desc + (uint64_t)((st * kTileBytes + ks * 32) >> 4), q_desc + (uint64_t)((ks * 32) >> 4),
                               kIdesc, ks > 0 ? 1u : 0u, leader);
                umma_commit(&slot_empty[st], leader);
                umma_commit(&s_full[sb], leader);  // (last: nothing of this thread is under way once the tile is known to be done)
            }
        }
        __syncwarp();
    } else if (warp == 6) {
        // ---------------- issuer of O^T += V^T . Pp^T ----------------
        const uint32_t leader = elect_one();
        const uint64_t v_desc = smem_desc(smem_u32(smem), 16, 1024, 2);  // MN-major: 8-key groups 1 KB apart
        const uint64_t p_desc = smem_desc(smem_u32(smem + kOffP), 16, 1024, 2);
        constexpr uint32_t kIdesc = idesc8<kInt>(0, 1, kN);
        int t = 0;
        for (; more && ok; ++x.b, more = x.load(p, plan, span)) {
            const int n = x.tiles();
            for (int i = 0; i < n && ok; ++i, ++t) {
                const int fill = 2 * t + 1, st = fill % kSlots, pb = t & 1;
                ok = mbar_wait(&slot_full[st], (uint32_t)(fill / kSlots) & 1u, abort_flag);
                if (ok) ok = mbar_wait(&p_full[pb], (uint32_t)(t >> 1) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t add = fresh[pb] ? 0u : 1u;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma8<kInt>(tmem + kColO, v_desc + (uint64_t)((st * kTileBytes + ks * 32 * kRowBytes) >> 4),
                               p_desc + (uint64_t)((pb * kN * kRowBytes + ks * 32) >> 4), kIdesc, ks > 0 ? 1u : add, leader);
                umma_commit(&slot_empty[st], leader);
                umma_commit(&p_empty[pb], leader);
            }
        }
        __syncwarp();
    } else if (warp < 4) {
        // ---------------- softmax: a thread per key; at a piece's end a thread per dim ----------------
        // (These warps meet at barriers: one whose wait has run out goes on to the end, where every later wait gives up at
        // once, rather than leave the others waiting.)
        HeadState *hs = reinterpret_cast<HeadState *>(smem + kOffHead);
        float2 *red = reinterpret_cast<float2 *>(smem + kOffRed);
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        // q's largest element is brought to 2^22 (int: digits of -128 to 127) or 2^8 (e4m3)
        constexpr int kQTop = kInt ? 22 : 8;
        // weights: 2^30 (int) or 2^7 (e4m3) at the reference, twice that at most
        constexpr float kWUnit = kInt ? 1073741824.0f : 128.0f;
        int t = 0;
        for (; more; ++x.b, more = x.load(p, plan, span)) {
            // ---- q in pieces: a warp per head, four elements a lane ----
            for (int h = warp; h < kHeads; h += 4) {
                float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (h < heads && lane * 4 < dim) {
                    const uint16_t *src = static_cast<const uint16_t *>(p.q) + (long long)x.b * p.q_row_stride +
                                          (long long)(head0 + h) * dim + lane * 4;
                    const uint2 raw = *reinterpret_cast<const uint2 *>(src);
                    const uint32_t v[2] = {raw.x, raw.y};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t u = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                        q[e] = p.q_bf16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
                    }
                }
                float top = fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3])));
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= !(fabsf(q[e]) < INFINITY);
                odd = __any_sync(0xffffffffu, odd);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                int ex = (int)(__float_as_uint(top) >> 23) - 127;  // 2^ex <= top < 2^(ex + 1)
                if (ex < -100 || odd) ex = -100;                    // (zero heads; odd ones become NaN by their factor)
                const float up = power2(kQTop - 1 - ex), down = power2(ex - kQTop + 1);
                uint32_t bytes[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = odd ? 0.0f : q[e] * up;
                    if (kInt) {
                        const int i = __float2int_rn(v);  // |i| <= 2^22, in three signed digits of 8 bits
                        const int lo = (int)(int8_t)(i & 255), i1 = (i - lo) >> 8, mid = (int)(int8_t)(i1 & 255), hi = (i1 - mid) >> 8;
                        bytes[0][e] = hi & 255, bytes[1][e] = mid & 255, bytes[2][e] = lo & 255;
                    } else {
#pragma unroll
                        for (int k = 0; k < 3; ++k) {
                            const __nv_fp8_storage_t c = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
                            bytes[k][e] = c;
                            const __half_raw back = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
                            v = (v - __half2float(*reinterpret_cast<const __half *>(&back))) * 16.0f;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const uint32_t n = k * kHeads + h;
                    uint8_t *row = smem + kOffQ;
                    *reinterpret_cast<uint32_t *>(row + swizzled(n, lane * 4)) =
                        bytes[k][0] | (bytes[k][1] << 8) | (bytes[k][2] << 16) | (bytes[k][3] << 24);
                }
                if (lane == 0) {
                    HeadState s;
                    s.factor = odd ? __uint_as_float(0x7fffffffu) : p.scale_log2 * down * (h < heads ? 1.0f : 0.0f);
                    s.slope = p.is_alibi ? exp2f(-8.0f * (float)(head0 + h + 1) / (float)p.head_q) * kLog2e : 0.0f;
                    s.m = s.mw = -FLT_MAX;
                    s.g = 1.0f;
                    hs[h] = s;
                }
            }
            fence_proxy_async();
            mbar_arrive(q_full);
            named_bar_sync(2, kSoftmaxThreads);  // the heads' states are there

            float l[kHeads], o[kHeads];
#pragma unroll
            for (int h = 0; h < kHeads; ++h) l[h] = o[h] = 0.0f;
            bool odd_v = false;   // a V scale is not a number
            int since = 0;        // tiles in the accumulator
            const int n = x.tiles();
            // cache row of this thread's key in tile i, or -1; and its scales, a tile ahead
            auto row_of = [&](int i) -> int {
                if (i >= n) return -1;
                const int key = x.key(p, i) + tid;
                if (key >= x.end) return -1;
                long long row;
                if (p.block_table) {
                    const int block = key >> p.page_shift;
                    if (block >= p.table_blocks) return -1;
                    const int page = p.block_table[(long long)x.b * p.table_stride + block];
                    row = page < 0 ? -1 : ((long long)page << p.page_shift) + (key & ((1 << p.page_shift) - 1));
                } else {
                    row = (long long)x.start + key;
                }
                return row >= 0 && row < p.rows ? (int)row : -1;
            };
            int row = row_of(0), row_next = row_of(1);
            float ks = row >= 0 ? p.k_scale[(long long)row * p.head_k + head_k] : 0.0f;
            float vs = row >= 0 ? p.v_scale[(long long)row * p.head_k + head_k] : 0.0f;
            // What the tensor core holds, in fp32 and in units of 2^mw: four pieces a head.
            auto accumulated = [&](float (&sum)[kHeads]) {
                uint32_t r[kN];
                tmem_ld16(lanes + kColO, r);
                tmem_wait_ld();
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    if (kInt) {
                        const float hi = fmaf((float)(int)r[h], 256.0f, (float)(int)r[kHeads + h]);
                        const float lo = fmaf((float)(int)r[2 * kHeads + h], 256.0f, (float)(int)r[3 * kHeads + h]);
                        sum[h] = fmaf(hi, 65536.0f, lo) * (1.0f / kWUnit);
                    } else {
                        const float hi = fmaf(__uint_as_float(r[kHeads + h]), 1.0f / 16, __uint_as_float(r[h]));
                        const float lo = fmaf(__uint_as_float(r[3 * kHeads + h]), 1.0f / 16, __uint_as_float(r[2 * kHeads + h]));
                        sum[h] = fmaf(lo, 1.0f / 256, hi) * (1.0f / kWUnit);
                    }
                }
            };

            for (int i = 0; i < n; ++i, ++t) {
                const int sb = t & 1, key0 = x.key(p, i);
                const bool valid = row >= 0;
                const float pos = (float)(key0 + tid - (x.len - 1));
                const float my_ks = ks, my_vs = vs;
                // the next tile's scales and the row after that
                row = row_next;
                row_next = row_of(i + 2);
                ks = row >= 0 ? p.k_scale[(long long)row * p.head_k + head_k] : 0.0f;
                vs = row >= 0 ? p.v_scale[(long long)row * p.head_k + head_k] : 0.0f;
                if (valid) odd_v |= !(my_vs < INFINITY);
                const float lv = __log2f(my_vs);

                ok &= (bool)__all_sync(0xffffffffu, mbar_wait(&s_full[sb], (uint32_t)(t >> 1) & 1u, abort_flag));
                tc_fence_after();
                float s[kHeads];
                {
                    uint32_t r[kN];
                    tmem_ld16(lanes + sb * kN, r);
                    tmem_wait_ld();
                    tc_fence_before();
                    mbar_arrive(&s_empty[sb]);
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        if (kInt)
                            s[h] = fmaf(int_to_float(r[h]), 65536.0f, fmaf(int_to_float(r[kHeads + h]), 256.0f, int_to_float(r[2 * kHeads + h])));
                        else
                            s[h] = fmaf(__uint_as_float(r[2 * kHeads + h]), 1.0f / 256, fmaf(__uint_as_float(r[kHeads + h]), 1.0f / 16, __uint_as_float(r[h])));
                    }
                }
                bool grown = false;
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    const float4 st = *reinterpret_cast<const float4 *>(&hs[h]);  // factor, slope, m, mw
                    s[h] *= st.x * my_ks;
                    if (p.is_alibi) s[h] = fmaf(st.y, pos, s[h]);
                    if (!valid) s[h] = -INFINITY;
                    grown |= s[h] > st.z + kHeadroom || s[h] + lv > st.w + kHeadroom;
                }
                const bool move = vote_any(grown);
                bool restart = since == 0;
                if (move || (kInt && since == kFlushTiles)) {
                    // ---- the references move: largest score and weight of the tile, by head ----
                    float shrink[kHeads];
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        float a = s[h], c = s[h] + lv;
                        if (!(c < INFINITY)) c = -INFINITY;  // (NaN or infinite scales are dealt with apart)
#pragma unroll
                        for (int d = 16; d > 0; d >>= 1) {
                            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
                            c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, d));
                        }
                        if (lane == 0) red[warp * kHeads + h] = make_float2(a, c);
                    }
                    named_bar_sync(2, kSoftmaxThreads);
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        float a = hs[h].m, c = hs[h].mw;
                        const float m0 = a, mw0 = c;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 y = red[w * kHeads + h];
                            a = fmaxf(a, y.x);
                            c = fmaxf(c, y.y);
                        }
                        l[h] *= exp2f(m0 - a);
                        shrink[h] = exp2f(mw0 - fmaxf(c, a - kWeightReach));
                    }
                    named_bar_sync(2, kSoftmaxThreads);
                    if (tid < kHeads) {
                        float a = hs[tid].m, c = hs[tid].mw;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 y = red[w * kHeads + tid];
                            a = fmaxf(a, y.x);
                            c = fmaxf(c, y.y);
                        }
                        c = fmaxf(c, a - kWeightReach);
                        hs[tid].m = a;
                        hs[tid].mw = c;
                        hs[tid].g = exp2f(0.5f * (a - c));
                    }
                    if (since > 0) {  // the last contraction has finished: take over what it has
                        ok &= (bool)__all_sync(0xffffffffu, mbar_wait(&p_empty[(t - 1) & 1], (uint32_t)((t - 1) >> 1) & 1u, abort_flag));
                        tc_fence_after();
                        float sum[kHeads];
                        accumulated(sum);
                        tc_fence_before();
#pragma unroll
                        for (int h = 0; h < kHeads; ++h) o[h] += sum[h];
                    }
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) o[h] *= shrink[h];
                    restart = true;
                    since = 0;
                    named_bar_sync(2, kSoftmaxThreads);
                }
                // ---- weights, in pieces, as the other contraction's operand ----
                if (t >= 2) ok &= (bool)__all_sync(0xffffffffu, mbar_wait(&p_empty[sb], ((uint32_t)(t >> 1) & 1u) ^ 1u, abort_flag));
                uint8_t *pt = smem + kOffP + sb * kN * kRowBytes;
                const float w_vs = valid ? my_vs : 0.0f;
#pragma unroll
                for (int h = 0; h < kHeads; h += 2) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float pr = exp2f(s[h + e] - hs[h + e].m);
                        l[h + e] += pr;
                        w[e] = (pr * hs[h + e].g) * (w_vs * (hs[h + e].g * kWUnit));
                    }
                    if (kInt) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t bits = __float2uint_rn(w[e]);
                            pt[swizzled(h + e, tid)] = (uint8_t)(bits >> 24);
                            pt[swizzled(kHeads + h + e, tid)] = (uint8_t)(bits >> 16);
                            pt[swizzled(2 * kHeads + h + e, tid)] = (uint8_t)(bits >> 8);
                            pt[swizzled(3 * kHeads + h + e, tid)] = (uint8_t)bits;
                        }
                    } else {
                        __half2 v = __floats2half2_rn(w[0], w[1]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t c = e4m3x2(v);
                            pt[swizzled(k * kHeads + h, tid)] = (uint8_t)c;
                            pt[swizzled(k * kHeads + h + 1, tid)] = (uint8_t)(c >> 8);
                            if (k < 3) v = __hmul2(__hsub2(v, from_e4m3x2(c)), __half2half2(__float2half_rn(16.0f)));
                        }
                    }
                }
                if (!kInt && key0 + kKeys > x.end) {
                    // Behind the last key there may be anything in a page, NaN included: 0 * NaN is not 0.
                    const int fill = 2 * t + 1, st = fill % kSlots;
                    ok &= (bool)__all_sync(0xffffffffu, mbar_wait(&slot_full[st], (uint32_t)(fill / kSlots) & 1u, abort_flag));
                    if (!valid) {
                        uint4 *v_row = reinterpret_cast<uint4 *>(smem + st * kTileBytes + tid * kRowBytes);
#pragma unroll
                        for (int c = 0; c < 8; ++c) v_row[c] = make_uint4(0, 0, 0, 0);
                    }
                }
                if (tid == 0) fresh[sb] = restart ? 1 : 0;
                ++since;
                fence_proxy_async();
                mbar_arrive(&p_full[sb]);
            }

            // ---- end of the piece ----
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
                if (lane == 0) red[warp * kHeads + h].x = l[h];
            }
            if (__any_sync(0xffffffffu, odd_v) && lane == 0) red[warp * kHeads].y = __uint_as_float(0x7fffffffu);
            else if (lane == 0) red[warp * kHeads].y = 0.0f;
            ok &= (bool)__all_sync(0xffffffffu, mbar_wait(&p_empty[(t - 1) & 1], (uint32_t)((t - 1) >> 1) & 1u, abort_flag));
            tc_fence_after();
            {
                float sum[kHeads];
                accumulated(sum);
                tc_fence_before();
#pragma unroll
                for (int h = 0; h < kHeads; ++h) o[h] += sum[h];
            }
            named_bar_sync(2, kSoftmaxThreads);
            const bool whole = x.begin == 0 && x.end == x.len;
            const int d = tid;  // the dim of this thread's row of the accumulator
            const float odd = red[0].y + red[kHeads].y + red[2 * kHeads].y + red[3 * kHeads].y;
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
                if (h >= heads) break;
                const float sum = red[h].x + red[kHeads + h].x + red[2 * kHeads + h].x + red[3 * kHeads + h].x;
                // o is in units of 2^mw, the sum in units of 2^m
                const float v = (sum > 0.0f ? o[h] * (1.0f / sum) * (1.0f / hs[h].g) * (1.0f / hs[h].g) : (sum == 0.0f ? 0.0f : sum)) + odd;
                const long long out = (long long)x.b * p.head_q + head0 + h;
                const long long piece = (span * 2 + (x.begin == 0 ? 1 : 0)) * p.head_q + head0 + h;
                const float lse = sum == 0.0f ? -INFINITY : (hs[h].m + log2f(sum)) * kLn2;
                if (d < dim) {
                    if (whole && p.o) {
                        uint16_t *dst = static_cast<uint16_t *>(p.o) + (long long)x.b * p.o_row_stride + (long long)(head0 + h) * dim + d;
                        *dst = p.q_bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
                    } else {
                        (whole ? p.own_o + out * dim : p.part_o + piece * dim)[d] = v;
                    }
                }
                if (tid == 0) {
                    if (whole && p.o) {
                        if (p.lse) p.lse[out] = lse;
                    } else {
                        *(whole ? p.own_lse + out : p.part_lse + piece) = lse;
                    }
                }
            }
            named_bar_sync(2, kSoftmaxThreads);  // (red and the heads' states are written anew)
        }
    }

    if (!ok && lane == 0) atomicExch(status, kStatusWaitTimeout);
    if (stays_for_prefix(p)) pdl_wait();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <bool kInt>
cudaError_t launch_typed(const StreamParams &p, int dim, int *status, const CUtensorMap &tm_k, const CUtensorMap &tm_v, cudaStream_t s) {
    static thread_local uint64_t ready = 0;  // devices on which this thread has raised the kernel's shared-memory limit
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((ready >> dev) & 1u)) {
        e = cudaFuncSetAttribute(da_codes_kernel<kInt>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    count_launch();
    return launch_kernel(da_codes_kernel<kInt>, dim3(p.head_k, p.spans), kThreads, kSmemBytes, s, true, p, dim, status, tm_k, tm_v);
}

}  // namespace

int codes_ctas() { return kCtas; }
int codes_heads() { return kHeads; }

cudaError_t launch_codes(int dim, int kind, const StreamParams &p, int *status, const CUtensorMap &tm_k, const CUtensorMap &tm_v,
                         cudaStream_t s) {
    return kind == 2 ? launch_typed<true>(p, dim, status, tm_k, tm_v, s) : launch_typed<false>(p, dim, status, tm_k, tm_v, s);
}

}  // namespace da
