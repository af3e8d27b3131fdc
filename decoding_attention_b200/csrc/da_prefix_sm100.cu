// Attention of a whole batch over a prefix that its sequences share, on the sm_100a tensor cores.
//
// One query token per sequence makes decode attention a matrix-vector product; over a shared prefix the
// `group` query heads of ALL sequences that use a KV head are rows of one matrix:
//     S[rows x keys] = Q . K^T,   O = softmax(S) . V,   rows = batch * group
// so that a prefix of n keys is read once (4 n head_k dim bytes) instead of once per sequence, for 4 n dim flops a row.
// Bound: the tensor pipe, once a KV head has more than about 200 rows; HBM below.  Each 128 x 128 score tile also costs
// 16 384 exponentials, 1 024 cycles of the SM's special-function units -- as long as its two contractions take.
//
// One CTA per SM runs two independent softmax streams of 128 rows (a lane of TMEM and a thread per row, so no row
// reduction crosses threads): while the threads of one stream work on their scores, the tensor pipe works for the other.
// The streams are the two row tiles of a unit, which share every K and V tile; a unit with one row tile gives its streams
// the even and the odd key tiles instead, and each leaves a part of its own.
//   TMEM, 512 columns: S 2 x 128 | O 2 x dim | P of a stream over its S (dim 64: in columns of its own).
//   Shared memory: Q 2 x 128 rows, five 128-key slots that K and V tiles take in turn, all by TMA with the 128-byte swizzle.
//   Warps: 2 x 4 softmax, one producer, one that issues the contractions in the order
//   S_a(0) S_b(0) | P.V_a(t) S_a(t+1) P.V_b(t) S_b(t+1) | ...  (one thread issues them, and they execute in that order, so
//   S may follow the P.V that reads the P lying under it).
// The CTAs take equal runs of key tiles whatever the number of units; what a CTA has of a unit is a part (normalised fp32
// rows and their log-sum-exp), and the parts, with those of the sequences' own keys, are joined by
// da_stream_merge_kernel.  Where there are many own keys too, some CTAs get no run and end at once (prefix_run): the key
// stream then has their SMs.  The reference has no prefix sharing.
//
// Measured: 1 024 rows x 16 384 keys x 8 KV heads, dim 128, on all SMs: 72 us inside the kernel, 0.95 PFLOP/s.  A key tile of
// both streams takes 2.6 us, 4 900 cycles, where the contractions alone take 2 050, the exponentials 2 048 and the tiles' way
// from L2 to shared memory about 1 800.  Tried without gain: half the exponentials by a polynomial on the fma pipe; an issuer
// per stream; streams that take the pipe in turns; other orders of the waits; two threads a row (registers spill).
#include "da_internal.h"
#include "da_prefix.h"
#include "da_tcgen05.cuh"

namespace da {
namespace {

constexpr int kRows = 128, kKeys = 128;
constexpr int kBlockBytes = 128 * 128;  // [128 rows or keys][64 columns]
constexpr int kSlots = 5;
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 384;  // (warps 10 and 11 only fill up the third warpgroup)
constexpr float kRescaleThreshold = 8.0f;  // log2 of what a score may exceed the maximum by that the reference stands for
// The softmax weights are rounded to the type of V, which the instruction wants on both sides.  fp16: the reference is 2^-7
// of the largest weight, so that fp16's subnormal numbers begin at 2^-21 of it and not at 2^-14; the weights then reach
// 2^15.  (bf16 has fp32's range.)
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;

template <int N, bool kMore>
__device__ __forceinline__ void set_max_registers() {
    if (kMore) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D>
struct PrefixCfg {
    static constexpr int kBlocks = D / 64;
    static constexpr int kTileBytes = kBlocks * kBlockBytes;
    static constexpr int kOffSlots = 2 * kTileBytes;
    static constexpr int kOffBar = kOffSlots + kSlots * kTileBytes;
    // q_full, q_empty, slot_full / slot_empty[kSlots], s_full, p_full, pv_done, o_free [2 each]
    static constexpr int kNumBars = 2 + 2 * kSlots + 8;
    static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;
    static constexpr int kColS = 0, kColO = 256;
    static constexpr int kColP = D == 64 ? 384 : 0;   // 64 columns a stream
    static constexpr int kStrideP = D == 64 ? 64 : 128;
    static_assert(D == 64 || D == 128, "head dim");
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

// What a CTA has to do of one unit: key tiles [t0, t1).
struct Piece {
    int hk, pair, t0, t1;
    bool split;  // one row tile: the streams share it and take the key tiles in turn
    long long next;
    __device__ __forceinline__ bool load(const PrefixGrid &g, long long at, long long end) {
        if (at >= end) return false;
        const long long unit = at / g.key_tiles;
        hk = (int)(unit / g.pairs);
        pair = (int)(unit - (long long)hk * g.pairs);
        t0 = (int)(at - unit * g.key_tiles);
        const long long left = end - at;
        t1 = left < g.key_tiles - t0 ? t0 + (int)left : g.key_tiles;
        split = 2 * pair + 1 >= g.row_tiles;
        next = at + (t1 - t0);
        return true;
    }
    // steps: one score tile of one stream each
    __device__ __forceinline__ int steps() const { return split ? t1 - t0 : 2 * (t1 - t0); }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
da_prefix_kernel(const PrefixParams p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v) {
    using C = PrefixCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *q_s = smem, *slot_s = smem + C::kOffSlots;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kOffBar);
    uint64_t *q_full = bars, *q_empty = bars + 1;
    uint64_t *slot_full = bars + 2, *slot_empty = slot_full + kSlots;
    uint64_t *s_full = slot_empty + kSlots, *p_full = s_full + 2, *pv_done = p_full + 2, *o_free = pv_done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kNumBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&slot_full[s], 1);
            mbar_init(&slot_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], kRows);
            mbar_init(&pv_done[s], 1);
            mbar_init(&o_free[s], kRows);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();  // the kernel before this call's may still be running
    pdl_launch_dependents();

    PrefixGrid g = p.grid;
    if (g.own_cost) {
        const long long keys = (long long)p.cu_seq_k[p.batch] - p.cu_seq_k[0];
        g.cta_tiles = prefix_run(g, keys > 0 ? keys : 0);
    }
    const long long total = g.total;
    const long long begin = (long long)blockIdx.x * g.cta_tiles;
    const long long end = begin + g.cta_tiles < total ? begin + g.cta_tiles : total;
    // With ALiBi the scores grow towards the end of the prefix: walked back to front, the first tiles set the maxima.
    auto tile_of = [&](const Piece &x, int i) { return p.is_alibi ? x.t1 - 1 - i : x.t0 + i; };

    constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t kIdescQK = instr_desc(kFmt, 0, kRows, kKeys);
    constexpr uint32_t kIdescPV = instr_desc(kFmt, 1, kRows, D);
    bool ok = true;
    Piece x;

    // The softmax threads hold a row of 128 scores: registers move to them from the other warpgroup
    // (2 x 128 x 208 + 128 x 80 of the 384 x 168 that the block is launched with).
    if (warp >= kProducerWarp) {
    set_max_registers<80, false>();
    if (warp == kProducerWarp) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            tma_prefetch_desc(&tm_q);
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
        const int run = p.table && (1 << p.page_shift) < kKeys ? 1 << p.page_shift : kKeys;
        const uint32_t q_bytes = (uint32_t)(C::kBlocks * 128 * p.group * g.tile_seqs);
        // Row of a key; rows of a page that is not in the pool are fetched from in front of the map, i.e. as zeros.
        auto row_of = [&](int key) -> int {
            if (!p.table) return key;
            const int page = p.table[key >> p.page_shift];
            const long long row = ((long long)page << p.page_shift) + (key & ((1 << p.page_shift) - 1));
            return page < 0 || row >= p.rows ? -kKeys : (int)row;
        };
        int fill = 0;  // tiles staged so far, K and V counted apart
        int pieces = 0;
        for (long long at = begin; ok && x.load(g, at, end); at = x.next, ++pieces) {
            if (pieces > 0) ok = mbar_wait(q_empty, (uint32_t)(pieces - 1) & 1u, abort_flag);
            if (!ok) break;
            if (lane == 0) {
                const int tiles = x.split ? 1 : 2;
                mbar_arrive_expect_tx(q_full, q_bytes * tiles);
                for (int i = 0; i < tiles; ++i)
                    for (int kb = 0; kb < C::kBlocks; ++kb)
                        tma_load_tile_3d(q_s + i * C::kTileBytes + kb * kBlockBytes, &tm_q, kb * 64, x.hk * p.group,
                                         (2 * x.pair + i) * g.tile_seqs, q_full);
            }
            for (int i = 0; i < x.t1 - x.t0 && ok; ++i) {
                const int key0 = tile_of(x, i) * kKeys;
                const int keys = min(kKeys, p.prefix_len - key0);
                for (int kv = 0; kv < 2 && ok; ++kv, ++fill) {
                    const int st = fill % kSlots;
                    if (fill >= kSlots) ok = mbar_wait(&slot_empty[st], ((uint32_t)(fill / kSlots) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    uint8_t *dst = slot_s + st * C::kTileBytes;
                    // A packed prefix ends with its tensor map, whose engine fills what lies behind with zeros; behind the
                    // last key of a page there may be anything, NaN included, so that tile is copied row by row.
                    if (!p.table || keys == kKeys) {
                        if (lane == 0) {
                            mbar_arrive_expect_tx(&slot_full[st], C::kTileBytes);
                            for (int k0 = 0; k0 < kKeys; k0 += run) {
                                const int key = key0 + k0;
                                const int row = row_of(key);
                                for (int kb = 0; kb < C::kBlocks; ++kb)
                                    tma_load_tile_3d(dst + kb * kBlockBytes + k0 * 128, kv ? &tm_v : &tm_k, kb * 64, x.hk, row, &slot_full[st]);
                            }
                        }
                    } else {
                        const T *src = reinterpret_cast<const T *>(kv ? p.v : p.k) + (size_t)x.hk * p.dim;
                        const long long stride = kv ? p.v_row_stride : p.k_row_stride;
                        constexpr int kChunks = D / 8;
                        for (int c0 = lane; c0 < kKeys * kChunks; c0 += 32) {
                            const int r = c0 / kChunks, c = c0 % kChunks, key = key0 + r;
                            long long row = -1;
                            if (r < keys && c * 8 < p.dim) {
                                const int page = p.table[key >> p.page_shift];
                                row = page < 0 ? -1 : ((long long)page << p.page_shift) + (key & ((1 << p.page_shift) - 1));
                                if (row >= p.rows) row = -1;
                            }
                            cp_async16(dst + (c >> 3) * kBlockBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                                       src + (row >= 0 ? row * stride + c * 8 : 0), row >= 0 ? 16u : 0u);
                        }
                        cp_async_commit();
                        cp_async_wait<0>();
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&slot_full[st]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ---------------- issuer of both contractions ----------------
        const uint32_t leader = elect_one();
        const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, 1024, 2);               // K-major, 8-row groups 1 KB apart
        const uint64_t k_desc = smem_desc(smem_u32(slot_s), 16, 1024, 2);
        const uint64_t v_desc = smem_desc(smem_u32(slot_s), kBlockBytes, 1024, 2);   // MN-major: 64-column blocks LBO apart
        int base = 0;              // key tiles of earlier pieces
        uint32_t done[2] = {0, 0}; // steps of each stream in earlier pieces
        int pieces = 0;
        uint32_t opened[2] = {0, 0};  // pieces in which the stream had a step
        for (long long at = begin; ok && x.load(g, at, end); at = x.next, ++pieces) {
            const int steps = x.steps(), tiles = x.t1 - x.t0;
            ok = mbar_wait(q_full, (uint32_t)pieces & 1u, abort_flag);
            auto scores = [&](int j) {
                const int l = j & 1, fill = 2 * (base + (x.split ? j : j >> 1)), st = fill % kSlots;
                ok = mbar_wait(&slot_full[st], (uint32_t)(fill / kSlots) & 1u, abort_flag);
                if (!ok) return;
                tc_fence_after();
                const uint64_t qd = q_desc + (uint64_t)((x.split ? 0 : l) * C::kTileBytes >> 4);
                const uint64_t kd = k_desc + (uint64_t)(st * C::kTileBytes >> 4);
#pragma unroll
                for (int kb = 0; kb < C::kBlocks; ++kb)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        umma_ss(tmem + C::kColS + l * kKeys, qd + (uint64_t)((kb * kBlockBytes + ks * 32) >> 4),
                                kd + (uint64_t)((kb * kBlockBytes + ks * 32) >> 4), kIdescQK, (kb | ks) ? 1u : 0u, leader);
                umma_commit(&s_full[l], leader);
                if (x.split || l == 1) umma_commit(&slot_empty[st], leader);
                if (j == steps - 1) umma_commit(q_empty, leader);
            };
            if (ok) scores(0);
            if (ok && steps > 1) scores(1);
            for (int j = 0; j < steps && ok; ++j) {
                const int l = j & 1, fill = 2 * (base + (x.split ? j : j >> 1)) + 1, st = fill % kSlots;
                ok = mbar_wait(&p_full[l], (done[l] + (uint32_t)(j >> 1)) & 1u, abort_flag);
                if (ok) ok = mbar_wait(&slot_full[st], (uint32_t)(fill / kSlots) & 1u, abort_flag);
                if (ok && j < 2 && opened[l] > 0) ok = mbar_wait(&o_free[l], (opened[l] - 1) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = v_desc + (uint64_t)(st * C::kTileBytes >> 4);
#pragma unroll
                for (int ks = 0; ks < kKeys / 16; ++ks)
                    umma_ts(tmem + C::kColO + l * D, tmem + C::kColP + l * C::kStrideP + ks * 8,
                            vd + (uint64_t)((ks * 16 * 128) >> 4), kIdescPV, (j >= 2 || ks > 0) ? 1u : 0u, leader);
                if (x.split || l == 1) umma_commit(&slot_empty[st], leader);
                umma_commit(&pv_done[l], leader);  // (last: what the threads wait for before the block ends)
                if (j + 2 < steps) scores(j + 2);
            }
            base += tiles;
            done[0] += (uint32_t)((steps + 1) / 2);
            done[1] += (uint32_t)(steps / 2);
            ++opened[0];
            if (steps > 1) ++opened[1];
        }
        __syncwarp();
    }
    } else {
        set_max_registers<208, true>();
        // ---------------- softmax and epilogue: a thread per row of a stream ----------------
        const int l = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_col = lanes + C::kColS + l * kKeys, o_col = lanes + C::kColO + l * D;
        const uint32_t p_col = lanes + C::kColP + l * C::kStrideP;
        uint32_t done = 0;  // score tiles of this stream so far
        for (long long at = begin; ok && x.load(g, at, end); at = x.next) {
            const int b = (2 * x.pair + (x.split ? 0 : l)) * g.tile_seqs + r / p.group;
            const int h = x.hk * p.group + r % p.group;
            const bool valid = r < p.group * g.tile_seqs && b < p.batch;
            const float slope = p.is_alibi ? exp2f(-8.0f * (float)(h + 1) / (float)p.head_q) * kLog2e : 0.0f;
            const int n = x.split ? (x.t1 - x.t0 + 1 - l) / 2 : x.t1 - x.t0;
            float m = -INFINITY, sum = 0.0f;
            for (int i = 0; i < n; ++i, ++done) {
                const int key0 = tile_of(x, x.split ? 2 * i + l : i) * kKeys;
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[l], done & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_col + c * 32, s[c]);
                tmem_wait_ld();
                float scale = p.scale_log2;
                if (p.is_alibi) {
                    // the bias is taken relative to the last key of the prefix, where it is small and matters
                    scale = 1.0f;
                    const float first = (float)(key0 - (p.prefix_len - 1));
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            s[c][j] = __float_as_uint(fmaf(slope, first + (float)(c * 32 + j), __uint_as_float(s[c][j]) * p.scale_log2));
                }
                if (key0 + kKeys > p.prefix_len) {
                    const int keys = p.prefix_len - key0;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c * 32 + j >= keys) s[c][j] = 0xff800000u;
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int j = 1; j < 32; ++j) top[c] = fmaxf(top[c], __uint_as_float(s[c][j]));
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
                const bool raise = valid && mx > m + (kRescaleThreshold + kLift<T>);
                if (__any_sync(0xffffffffu, raise)) {
                    float shrink = 1.0f;
                    if (raise) {
                        shrink = exp2f(m - (mx - kLift<T>));  // 0 on the first tile
                        m = mx - kLift<T>;
                        sum *= shrink;
                    }
                    if (i > 0) {  // the accumulator is idle once the last P.V of this stream has finished
                        ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[l], (done - 1) & 1u, abort_flag));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(o_col + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                            tmem_st32(o_col + c * 32, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;  // (a row whose scores are all -inf so far)
                float part[2] = {0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float p0 = exp2f(fmaf(__uint_as_float(s[2 * c + (j >> 4)][2 * (j & 15)]), scale, -ref));
                        const float p1 = exp2f(fmaf(__uint_as_float(s[2 * c + (j >> 4)][2 * (j & 15) + 1]), scale, -ref));
                        part[0] += p0;
                        part[1] += p1;
                        if (std::is_same<T, __nv_bfloat16>::value) {
                            const __nv_bfloat162 y = __floats2bfloat162_rn(p0, p1);
                            w[j] = *reinterpret_cast<const uint32_t *>(&y);
                        } else {
                            const __half2 y = __floats2half2_rn(p0, p1);
                            w[j] = *reinterpret_cast<const uint32_t *>(&y);
                        }
                    }
                    tmem_st32(p_col + c * 32, w);
                }
                sum += part[0] + part[1];
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[l]);
            }
            if (!ok) break;
            // ---- the part of this piece ----
            const long long unit = (long long)x.hk * g.pairs + x.pair;
            const long long first_cta = unit * g.key_tiles / g.cta_tiles;
            const int part = (int)(blockIdx.x - first_cta) * (x.split ? 2 : 1) + (x.split ? l : 0);
            const size_t row = ((size_t)part * p.batch + (valid ? b : 0)) * p.head_q + h;
            if (n > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[l], (done - 1) & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
                float *dst = p.part_o + row * p.dim;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(o_col + c * 32, o);
                    tmem_wait_ld();
                    if (!valid || c * 32 >= p.dim) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        *reinterpret_cast<float4 *>(dst + c * 32 + 4 * j) =
                            make_float4(__uint_as_float(o[4 * j]) * inv, __uint_as_float(o[4 * j + 1]) * inv,
                                        __uint_as_float(o[4 * j + 2]) * inv, __uint_as_float(o[4 * j + 3]) * inv);
                }
                tc_fence_before();
                mbar_arrive(&o_free[l]);
            }
            if (valid) {
                float lse = -INFINITY;
                if (n > 0 && sum != 0.0f) {
                    // positions count back from the sequence's last key, which lies len - 0 keys behind the prefix's
                    const float shift = p.is_alibi ? -slope * (float)(p.cu_seq_k[b + 1] - p.cu_seq_k[b]) : 0.0f;
                    lse = (m + log2f(sum) + shift) * kLn2;
                }
                p.part_lse[row] = lse;
            }
        }
    }

    if (!ok && lane == 0) atomicExch(p.status, kStatusWaitTimeout);
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int D>
cudaError_t launch_typed(const PrefixParams &p, const CUtensorMap &tm_q, const CUtensorMap &tm_k, const CUtensorMap &tm_v,
                         cudaStream_t s) {
    using C = PrefixCfg<D>;
    static thread_local uint64_t ready = 0;  // devices on which this thread has raised the kernel's shared-memory limit
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((ready >> dev) & 1u)) {
        e = cudaFuncSetAttribute(da_prefix_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    count_launch();
    return launch_kernel(da_prefix_kernel<T, D>, dim3(p.grid.ctas), kThreads, C::kSmemBytes, s, true, p, tm_q, tm_k, tm_v);
}

}  // namespace

cudaError_t launch_prefix(bool bf16, const PrefixParams &p, const CUtensorMap &tm_q, const CUtensorMap &tm_k,
                          const CUtensorMap &tm_v, cudaStream_t s) {
    if (p.dim == 64)
        return bf16 ? launch_typed<__nv_bfloat16, 64>(p, tm_q, tm_k, tm_v, s) : launch_typed<__half, 64>(p, tm_q, tm_k, tm_v, s);
    // (dim 96 runs on 128 columns: its tensor maps end at column 96 and the rest arrives as zeros)
    return bf16 ? launch_typed<__nv_bfloat16, 128>(p, tm_q, tm_k, tm_v, s) : launch_typed<__half, 128>(p, tm_q, tm_k, tm_v, s);
}

}  // namespace da
