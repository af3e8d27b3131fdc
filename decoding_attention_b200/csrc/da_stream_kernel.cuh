// Decode attention as one stream of keys, for caches of 8- and 4-bit codes with a scale per (token, KV head) -- and
// for 16-bit caches, where it serves the sequences' own keys behind a shared prefix.
//
//     s_j = c ks_j (q . kc_j) [+ slope (j - (len - 1))],   o = sum_j softmax(s)_j vs_j vc_j
//
// Bound: HBM for 16-bit rows (0.95 of the copy rate next to a prefix); the issue slots for codes.  A byte of a quantised
// cache carries one or two elements, each of which becomes an operand of one multiply-add per query head and has to be
// converted first: at the HBM rate 23 bytes a clock reach an SM, which is more than its CUDA cores can convert to fp32 and
// multiply.  So the codes are turned into fp16 PAIRS (exact for all three
// formats: byte and nibble pairs by one logic operation into the mantissa of 1024 and one subtraction, e4m3 by the
// hardware's pair conversion) straight in the registers in which mma.sync wants them, with the KEYS (and for the second
// product the DIMS) as the 16 rows of a tile and the query heads as its 8 columns:
//     S^T[16 keys x 8 heads] = K[16 x D] . Q^T,      O^T[D x 8 heads] += V^T[D x 16] . P^T
// The products' reduction index may be permuted freely, so a lane loads its elements with 16-byte accesses of
// untransposed rows, and the transposition of V is two byte permutes per pair of keys.  S^T becomes P^T by one movmatrix
// per 8 keys.  16 keys of 128 columns and eight heads take 434 (int4), 462 (e4m3) and 589 (int8) instructions, all told:
// 4 x 65 536 keys with 64 over 8 heads come to 89 us (int4, HBM time 44), 102 (e4m3, 85) and 118 us (int8, 85).
//
// For 8-bit codes and groups of up to four heads da_codes_sm100.cu, where the codes themselves are tensor-core operands, is
// faster.  Tried for the rest and left out: the codes widened to fp16 in shared memory by warps of their own, once a key, as
// tcgen05 operands (the chain of widening, scores, weights and the other contraction takes 3 000 cycles a tile with the one
// CTA an SM that fits: 191 us for the int4 case above); and 32 heads a warp, so that a group of 32 is widened once instead
// of twice (128 sequences of 2 048 int4 keys, 32 heads over one KV head: 51 us against 42 with two warps of 16 heads; 44 now).
//
// And the weights below as two fp16 parts, 22 bits, by a second multiply-add each: 128 sequences of 2 048 int4 keys, 32 heads,
// 48 us instead of 43.
//
// q is brought to fp16 with a power of two per head that makes its largest element 1..2, undone in the score's factor:
// exact, but for elements of a bf16 head below 2^-14 of its largest, which keep 2^-25 of that.  The weights w_j = p_j vs_j
// are rounded to fp16 in units of their own, one factor per head that is kept like the reference maximum: the largest
// weight so far comes to 2^7..2^15, so that a weight is off by half a step, 2^-11 of itself, or by 2^-32 of the largest.
// Where it sets the units the largest is not rounded at all, which takes the error of fp16 outputs from 1.4 to 1.1 times their
// own rounding.  (The units follow the weights and not the probabilities: a key that leads by far may have a V row of zeros.)  16-bit
// caches: the weights are the probabilities, rounded to the cache's type, which V has and the instruction wants on both
// sides.  Between q and o these are the only roundings to fewer bits; sums, maxima and outputs are fp32.
//
// Work split.  Lengths live on the device, so the CTAs cut the concatenated keys of the whole batch into equal spans
// (StreamParams): any mix of lengths keeps all SMs busy to the end, without a sort or a guess of the longest sequence.
// A sequence inside one span is finished by its CTA; the pieces of the others are joined by da_stream_merge_kernel,
// which also writes the rows of empty sequences.  Eight warps a CTA: `head_warps` (KV head, head chunk) streams, so that
// the CTA reads whole rows of the cache, x `key_warps` interleaved parts of the keys.  Every warp has its own ring of
// tiles (cp.async, zero fill for rows that are masked or that no page holds), filled across the ends of sequences.
#pragma once

#include <cfloat>

#include "da_internal.h"
#include "da_stream.h"

namespace da {

constexpr int kStreamWarps = 8;

// What a cache element is: 0 fp16, 1 FP8 e4m3, 2 int8, 3 int4, 4 bf16.
template <int KIND, int D, int NT_>
struct StreamCfg {
    static constexpr bool kQuant = KIND >= 1 && KIND <= 3;
    static constexpr int NT = NT_;
    static constexpr int RB = KIND == 3 ? D / 2 : (kQuant ? D : 2 * D);  // bytes of a row
    static constexpr int EPW = KIND == 3 ? 8 : (kQuant ? 4 : 2);        // elements of a 4-byte word
    static constexpr int TK = RB >= 96 ? 16 : 32;                        // keys of a tile
    static constexpr int KSTEPS = D / 16, MTILES = D / 16;
    static constexpr int KW = RB / 16;                     // words of a K row in a lane (a quarter of the row)
    static constexpr int VW = (RB + 31) / 32;              // words of a V row in a lane (an eighth; the last may be half)
    static constexpr int CPR = RB / 16;                    // 16-byte chunks of a row
    static_assert(TK * CPR % 32 == 0, "all lanes take part in every copy of a tile");
    static constexpr int kScaleBytes = kQuant ? TK * 8 : 0;
    static constexpr int kStageBytes = 2 * TK * RB + kScaleBytes;
    static constexpr bool kTwoCtas = D <= 128 && NT == 1 && RB <= 128;
    static constexpr int kMergeRow = D + 4;                // floats of a head's record in the merge area
    static constexpr int kMergeBytes = kStreamWarps / 2 * NT * 8 * kMergeRow * 4;
    static constexpr int kBudget = (kTwoCtas ? 113 : 226) * 1024 - kMergeBytes - 1024;
    static constexpr int kFit = kBudget / kStreamWarps / kStageBytes;
    static constexpr int STAGES = kFit > 6 ? 6 : kFit;
    static_assert(STAGES >= 2, "a ring needs two stages");
    static constexpr int kSmemBytes = kStreamWarps * STAGES * (kStageBytes + 4) + kMergeBytes + 16;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
    if (bf16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit values held two a lane.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void cp_async4(void *dst_smem, const void *src_gmem, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst_smem)), "l"(src_gmem), "r"(src_bytes)
                 : "memory");
}
__device__ __forceinline__ void cp_async16_full(void *dst_smem, const void *src_gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst_smem)), "l"(src_gmem) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The power of two at or below a positive number (-127: none that is normal), and back.
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
constexpr int kMostScaled = 100;  // log2 of what a V scale may come to in the units of the weights

// ---- codes to pairs of fp16 --------------------------------------------------------------------
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b),
                              *reinterpret_cast<const __half2 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Bytes 0 and 2 of x, signed: 1024 + 128 + value is an fp16 whose mantissa is the byte with its sign flipped.
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) { return h2_sub((x & 0x00ff00ffu) ^ 0x64806480u, 0x64806480u); }
// Nibbles 0 and 4 of x, signed: 1024 + 8 + value.
__device__ __forceinline__ uint32_t int4_pair_low(uint32_t x) { return h2_sub((x & 0x000f000fu) ^ 0x64086408u, 0x64086408u); }
// Nibbles 1 and 5: 1024 + 16 (8 + value), divided by 16 in the fma (1 / 16, -72).
__device__ __forceinline__ uint32_t int4_pair_high(uint32_t x) {
    return h2_fma((x & 0x00f000f0u) ^ 0x64806480u, 0x2c002c00u, 0xd480d480u);
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t x) {  // the low two bytes
    uint32_t y;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(y) : "r"(x));
    return y;
}

// The two A registers that one K row gives to reduction step `step` from a lane's words, and the element (0 .. EPW-1 of
// word, or of two words) that each half holds: see stream_pair_elem.
template <int KIND, int N>
__device__ __forceinline__ void k_pairs(const uint32_t (&w)[N], int step, uint32_t &p0, uint32_t &p1) {
    if (KIND == 3) {
        const uint32_t x = w[step >> 1] >> ((step & 1) * 8);
        p0 = int4_pair_low(x);
        p1 = int4_pair_high(x);
    } else if (KIND == 2) {
        p0 = int8_pair(w[step]);
        p1 = int8_pair(w[step] >> 8);
    } else if (KIND == 1) {
        p0 = e4m3_pair(w[step]);
        p1 = e4m3_pair(w[step] >> 16);
    } else {
        p0 = w[2 * step];
        p1 = w[2 * step + 1];
    }
}
// (first, second) element of A register `reg` of step `step`, counted from the start of the step's word(s).
template <int KIND>
__device__ __forceinline__ constexpr int pair_elem(int step, int reg, int half) {
    if (KIND == 3) return 2 * (step & 1) + reg + 4 * half;
    if (KIND == 2) return reg + 2 * half;
    return 2 * reg + half;
}
// V words of two keys -> pairs (key a, key b) of the word's elements in order.
template <int KIND, int N>
__device__ __forceinline__ void v_pairs(uint32_t a, uint32_t b, uint32_t (&p)[N]) {
    if (KIND == 3) {
#pragma unroll
        for (int h = 0; h < N / 4; ++h) {
            const uint32_t x = __byte_perm(a, b, h ? 0x7632 : 0x5410);
            p[4 * h] = int4_pair_low(x);
            p[4 * h + 1] = int4_pair_high(x);
            p[4 * h + 2] = int4_pair_low(x >> 8);
            p[4 * h + 3] = int4_pair_high(x >> 8);
        }
    } else if (KIND == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t x = __byte_perm(a, b, h ? 0x7632 : 0x5410);
            p[2 * h] = int8_pair(x);
            p[2 * h + 1] = int8_pair(x >> 8);
        }
    } else if (KIND == 1) {
        const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
        p[0] = e4m3_pair(x);
        p[1] = e4m3_pair(x >> 16);
        p[2] = e4m3_pair(y);
        p[3] = e4m3_pair(y >> 16);
    } else {
        p[0] = __byte_perm(a, b, 0x5410);
        p[1] = __byte_perm(a, b, 0x7632);
    }
}

// Byte offset, in an unswizzled row, of word w of lane part c (K: four parts) or r (V: eight parts): pieces of 16 bytes
// while they last, then one each of 8, 4 and (V) 2 bytes.
template <int RB, int PARTS>
__device__ __forceinline__ constexpr int word_offset(int w, int part) {
    constexpr int n16 = RB / (16 * PARTS);
    if (w < 4 * n16) return (w / 4 * PARTS + part) * 16 + w % 4 * 4;
    int base = n16 * 16 * PARTS;
    w -= 4 * n16;
    if ((RB - base) >= 8 * PARTS) {
        if (w < 2) return base + part * 8 + w * 4;
        base += 8 * PARTS;
        w -= 2;
    }
    if ((RB - base) >= 4 * PARTS) {
        if (w < 1) return base + part * 4;
        base += 4 * PARTS;
        w -= 1;
    }
    return base + part * 2;
}

// Where a 16-byte chunk of a staged row lies: permuted so that the lanes of one access hit different banks (a phase of
// K's loads reads two rows that differ in bit 2, one of V's four rows that differ in bits 0 and 1).
template <int RB>
__device__ __forceinline__ int k_chunk(int row, int chunk) {
    return RB % 128 == 0 ? chunk ^ (row & 4) : chunk;
}
template <int RB>
__device__ __forceinline__ int v_chunk(int row, int chunk) {
    return RB % 128 == 0 ? chunk ^ (2 * (row & 3)) : (RB == 64 ? chunk ^ (row & 2) : chunk);
}

template <int RB>
__device__ __forceinline__ void load_k_words(const uint8_t *tile, int row, int c, uint32_t (&w)[RB / 16]) {
    const uint8_t *base = tile + row * RB;
    constexpr int n16 = RB / 64;
#pragma unroll
    for (int i = 0; i < n16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4 *>(base + k_chunk<RB>(row, i * 4 + c) * 16);
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
    }
    if (RB & 32) {
        const uint2 x = *reinterpret_cast<const uint2 *>(base + n16 * 64 + c * 8);
        w[4 * n16] = x.x, w[4 * n16 + 1] = x.y;
    }
    if (RB & 16) w[RB / 16 - 1] = *reinterpret_cast<const uint32_t *>(base + RB - 16 + c * 4);
}
template <int RB>
__device__ __forceinline__ void load_v_words(const uint8_t *tile, int row, int r, uint32_t (&w)[(RB + 31) / 32]) {
    const uint8_t *base = tile + row * RB;
    constexpr int n16 = RB / 128;
#pragma unroll
    for (int i = 0; i < n16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4 *>(base + v_chunk<RB>(row, i * 8 + r) * 16);
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
    }
    constexpr int b8 = n16 * 128, i8 = n16 * 4;
    if (RB & 64) {
        const int at = b8 + r * 8;
        const uint2 x = *reinterpret_cast<const uint2 *>(base + v_chunk<RB>(row, at >> 4) * 16 + (at & 15));
        w[i8] = x.x, w[i8 + 1] = x.y;
    }
    constexpr int b4 = b8 + (RB & 64), i4 = i8 + ((RB & 64) ? 2 : 0);
    if (RB & 32) w[i4] = *reinterpret_cast<const uint32_t *>(base + b4 + r * 4);
    constexpr int b2 = b4 + (RB & 32), i2 = i4 + ((RB & 32) ? 1 : 0);
    if (RB & 16) w[i2] = *reinterpret_cast<const uint16_t *>(base + b2 + r * 2);
}

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(kStreamWarps * 32, StreamCfg<KIND, D, NT>::kTwoCtas ? 2 : 1)
    da_stream_kernel(const StreamParams p) {
    using C = StreamCfg<KIND, D, NT>;
    constexpr int TK = C::TK, RB = C::RB, STAGES = C::STAGES, MT = TK / 16;
    constexpr bool kBf16 = KIND == 4;
    // fp16 weights (16-bit caches): the reference is 2^-7 of the largest, so that fp16's subnormal numbers begin at 2^-21 of
    // it and not at 2^-14; the weights then reach 2^15.  (bf16 has fp32's range.)
    constexpr float kLift = KIND == 0 ? 7.0f : 0.0f;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, c = lane & 3;
    uint8_t *ring = smem + warp * (STAGES * C::kStageBytes);
    uint32_t *masks = reinterpret_cast<uint32_t *>(smem + kStreamWarps * STAGES * C::kStageBytes) + warp * STAGES;
    float *merge = reinterpret_cast<float *>(smem + kStreamWarps * STAGES * (C::kStageBytes + 4));

    if (!p.chained) pdl_wait();  // the kernel before this call's may still be running
    pdl_launch_dependents();
    const bool stays = stays_for_prefix(p);
    const SpanPlan plan = span_plan(p);
    const long long span = blockIdx.x;
    if (span * plan.units >= plan.total) {
        if (stays) pdl_wait();
        return;
    }

    const int kpart = warp / p.head_warps;
    const int stream = blockIdx.y * p.head_warps + warp % p.head_warps;
    const bool idle = stream >= p.head_k * p.chunks;  // (these warps only keep the barriers company)
    const int head_k = idle ? 0 : stream / p.chunks;
    const int chunk = idle ? 0 : stream - head_k * p.chunks;
    const int head0 = head_k * p.group + chunk * 8 * NT;           // first query head of this warp
    const int heads = min(8 * NT, p.group - chunk * 8 * NT);       // how many it has
    const int stride = TK * p.key_warps;

    const uint8_t *kbase = static_cast<const uint8_t *>(p.k) + (long long)head_k * RB;
    const uint8_t *vbase = static_cast<const uint8_t *>(p.v) + (long long)head_k * RB;
    const long long kstep = KIND == 3 ? p.k_row_stride / 2 : p.k_row_stride * (C::kQuant ? 1 : 2);  // bytes
    const long long vstep = KIND == 3 ? p.v_row_stride / 2 : p.v_row_stride * (C::kQuant ? 1 : 2);

    PieceCursor con;
    con.b = find_sequence(plan, p.cu_seq_k, p.batch, span * plan.units, lane);
    bool more = con.load(p, plan, span);

    // ---- producer side: tiles in the order in which this warp will want them ----
    // Tiles that a piece has for this warp, and the first key of the i-th it takes.  With ALiBi the scores grow towards the
    // end of a sequence: walked back to front, the first tiles set the reference maxima for the rest.
    auto tiles_of = [&](const PieceCursor &x) {
        const int keys = x.end - x.begin - kpart * TK;
        return keys > 0 ? (keys + stride - 1) / stride : 0;
    };
    auto tile_key = [&](const PieceCursor &x, int i, int n) { return x.begin + kpart * TK + (p.is_alibi ? n - 1 - i : i) * stride; };
    PieceCursor pro = con;
    bool pro_more = more && !idle;
    int pro_at = 0, pro_n = pro_more ? tiles_of(pro) : 0, pro_key = 0;
    auto settle = [&]() {  // moves on to a piece that has a tile for this warp
        while (pro_more && pro_at >= pro_n) {
            ++pro.b;
            pro_more = pro.load(p, plan, span);
            pro_at = 0;
            pro_n = pro_more ? tiles_of(pro) : 0;
        }
        pro_key = tile_key(pro, pro_at, pro_n);
    };
    // The first cache row of the next tile if all its keys are there, one row behind the other; -1 otherwise.
    auto lookup = [&]() -> int {
        if (!pro_more || pro_key + TK > pro.end) return -1;
        long long row;
        if (p.block_table) {
            const int block = pro_key >> p.page_shift;
            if ((1 << p.page_shift) < TK || block >= p.table_blocks) return -1;
            const int page = p.block_table[(long long)pro.b * p.table_stride + block];
            row = page < 0 ? -1 : ((long long)page << p.page_shift) + (pro_key & ((1 << p.page_shift) - 1));
        } else {
            row = (long long)pro.start + pro_key;
        }
        return row >= 0 && row + TK <= p.rows ? (int)row : -1;
    };
    // Any other tile: the cache row of key pro_key + lane, or -1 (behind the end, outside the table, the pool or the cache).
    auto lookup_row = [&]() -> int {
        const int key = pro_key + lane;
        if (lane >= TK || key >= pro.end) return -1;
        long long row;
        if (p.block_table) {
            const int block = key >> p.page_shift;
            if (block >= p.table_blocks) return -1;
            const int page = p.block_table[(long long)pro.b * p.table_stride + block];
            row = page < 0 ? -1 : ((long long)page << p.page_shift) + (key & ((1 << p.page_shift) - 1));
        } else {
            row = (long long)pro.start + key;
        }
        return row >= 0 && row < p.rows ? (int)row : -1;
    };
    settle();
    int row_next = lookup();
    int fill = 0;
    constexpr uint32_t kAllKeys = TK == 32 ? 0xffffffffu : (1u << TK) - 1u;
    constexpr int kCopies = TK * C::CPR / 32;         // 16-byte copies of a lane for a K tile
    const int row_l = lane / C::CPR, chunk_l = lane % C::CPR;
    auto issue = [&]() {
        if (pro_more) {
            uint8_t *stage = ring + fill * C::kStageBytes;
            float *sc = reinterpret_cast<float *>(stage + 2 * TK * RB);
            if (row_next >= 0) {
                if (lane == 0) masks[fill] = kAllKeys;
                const uint8_t *ks = kbase + (long long)row_next * kstep, *vs = vbase + (long long)row_next * vstep;
                if (32 % C::CPR == 0) {
                    // copy i takes the rows 32 / CPR further: the lane's place in them stays the same
                    ks += (long long)row_l * kstep + chunk_l * 16;
                    vs += (long long)row_l * vstep + chunk_l * 16;
                    const long long ks_next = 32 / C::CPR * kstep, vs_next = 32 / C::CPR * vstep;
#pragma unroll
                    for (int i = 0; i < kCopies; ++i) {
                        const int tr = i * (32 / C::CPR) + row_l;
                        cp_async16_full(stage + tr * RB + k_chunk<RB>(tr, chunk_l) * 16, ks);
                        cp_async16_full(stage + TK * RB + tr * RB + v_chunk<RB>(tr, chunk_l) * 16, vs);
                        ks += ks_next;
                        vs += vs_next;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kCopies; ++i) {
                        const int idx = i * 32 + lane;
                        const int tr = idx / C::CPR, ch = idx - tr * C::CPR;
                        cp_async16_full(stage + tr * RB + k_chunk<RB>(tr, ch) * 16, ks + (long long)tr * kstep + ch * 16);
                        cp_async16_full(stage + TK * RB + tr * RB + v_chunk<RB>(tr, ch) * 16, vs + (long long)tr * vstep + ch * 16);
                    }
                }
                if (C::kQuant && lane < TK) {
                    const long long at = (long long)(row_next + lane) * p.head_k + head_k;
                    cp_async4(sc + lane, p.k_scale + at, 4u);
                    cp_async4(sc + TK + lane, p.v_scale + at, 4u);
                }
            } else {
                const int row = lookup_row();
                const unsigned valid = __ballot_sync(0xffffffffu, row >= 0);
                if (lane == 0) masks[fill] = valid;
#pragma unroll 1
                for (int idx = lane; idx < TK * C::CPR; idx += 32) {
                    const int tr = idx / C::CPR, ch = idx - tr * C::CPR;
                    const int src = __shfl_sync(0xffffffffu, row, tr);
                    const long long at = src >= 0 ? src : 0;
                    const uint32_t bytes = src >= 0 ? 16u : 0u;
                    cp_async16(stage + tr * RB + k_chunk<RB>(tr, ch) * 16, kbase + at * kstep + ch * 16, bytes);
                    cp_async16(stage + TK * RB + tr * RB + v_chunk<RB>(tr, ch) * 16, vbase + at * vstep + ch * 16, bytes);
                }
                if (C::kQuant && lane < TK) {
                    const long long at = (long long)(row >= 0 ? row : 0) * p.head_k + head_k;
                    cp_async4(sc + lane, p.k_scale + at, row >= 0 ? 4u : 0u);
                    cp_async4(sc + TK + lane, p.v_scale + at, row >= 0 ? 4u : 0u);
                }
            }
            fill = fill + 1 == STAGES ? 0 : fill + 1;
            ++pro_at;
            settle();
            row_next = lookup();
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue();

    int drain = 0;
    // physical keys of this lane's rows in S^T (r -> key_r, r + 8 -> 8 + key_r) and in V^T's reduction
    const int key_r = (r & 1) * 4 + ((r >> 1) ^ (r & 1));

    for (; more; ++con.b, more = con.load(p, plan, span)) {
        // ---- q of this piece as B operands ----
        uint32_t qf[C::KSTEPS][NT][2];
        float factor[NT][2], slope[NT][2];
        {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bool have = !idle && n * 8 + r < heads;
                const uint16_t *row = static_cast<const uint16_t *>(p.q) + (long long)con.b * p.q_row_stride +
                                      (long long)(head0 + (have ? n * 8 + r : 0)) * D;
                uint16_t h[C::KSTEPS][4];  // the lane's elements of the head's row, as the reduction steps want them
#pragma unroll
                for (int s = 0; s < C::KSTEPS; s += KIND == 3 ? 2 : 1) {
                    const int word = KIND == 3 ? s >> 1 : (C::kQuant ? s : 2 * s);
                    const uint16_t *src = row + word_offset<RB, 4>(word, c) * C::EPW / 4;
                    uint32_t v[4] = {0, 0, 0, 0};
                    if (have) {
                        if (KIND == 3) {
                            const uint4 y = *reinterpret_cast<const uint4 *>(src);
                            v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
                        } else {
                            const uint2 y = *reinterpret_cast<const uint2 *>(src);
                            v[0] = y.x, v[1] = y.y;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < (KIND == 3 ? 2 : 1); ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int el = pair_elem<KIND>(s + t, e >> 1, e & 1);
                            h[s + t][e] = (uint16_t)(v[el >> 1] >> (16 * (el & 1)));
                        }
                }
                float x[C::KSTEPS][4];
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < C::KSTEPS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (C::kQuant) {
                            x[s][e] = p.q_bf16 ? __uint_as_float((uint32_t)h[s][e] << 16) : __half2float(__ushort_as_half(h[s][e]));
                            top = fmaxf(top, fabsf(x[s][e]));
                        } else {
                            x[s][e] = __uint_as_float((uint32_t)h[s][e]);
                        }
                    }
                float up = 1.0f, f = p.scale_log2;
                if (C::kQuant) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // 2^-e and 2^e of the largest element; zeros, infinities and NaN stay as they are
                    const int ex = (int)(__float_as_uint(top) >> 23);
                    if (ex > 1 && ex < 255) {
                        const int e = min(ex, 253);  // (2^-e is a normal number then)
                        up = __uint_as_float((uint32_t)(254 - e) << 23);
                        f = p.scale_log2 * __uint_as_float((uint32_t)e << 23);
                    }
                }
#pragma unroll
                for (int s = 0; s < C::KSTEPS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (C::kQuant) {
                            const __half2 v = __floats2half2_rn(x[s][2 * h] * up, x[s][2 * h + 1] * up);
                            qf[s][n][h] = *reinterpret_cast<const uint32_t *>(&v);
                        } else {
                            qf[s][n][h] = __float_as_uint(x[s][2 * h]) | (__float_as_uint(x[s][2 * h + 1]) << 16);
                        }
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    factor[n][e] = __shfl_sync(0xffffffffu, f, 8 * c + 4 * e);
                    slope[n][e] = 0.0f;
                    if (p.is_alibi) slope[n][e] = exp2f(-8.0f * (head0 + n * 8 + 2 * c + e + 1) / p.head_q) * kLog2e;
                }
            }
        }
        float m[NT][2], l[NT][2], f[NT][2], acc[C::MTILES][NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) m[n][e] = -FLT_MAX, l[n][e] = 0.0f, f[n][e] = 1.0f;
#pragma unroll
        for (int t = 0; t < C::MTILES; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][n][e] = 0.0f;

        // Units of the weights: f a head, f_top the largest of this lane's heads.
        uint32_t unset = 0;  // heads whose reference maximum has risen, but no weight come since (a bit each, the same in a column's lanes)
        float f_top = 1.0f;
        auto set_f_top = [&]() {
            f_top = f[0][0];
#pragma unroll
            for (int n = 0; n < NT; ++n) f_top = fmaxf(f_top, fmaxf(f[n][0], f[n][1]));
        };

        const int tiles = idle ? 0 : tiles_of(con);
        for (int step = 0; step < tiles; ++step) {
            const int key0 = tile_key(con, step, tiles);
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            issue();
            const uint8_t *ktile = ring + drain * C::kStageBytes, *vtile = ktile + TK * RB;
            const float *sc = reinterpret_cast<const float *>(vtile + TK * RB);
            const uint32_t valid = masks[drain];
            drain = drain + 1 == STAGES ? 0 : drain + 1;

            // ---- scores ----
            float s[MT][NT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t w0[C::KW], w1[C::KW];
                load_k_words<RB>(ktile, t * 16 + key_r, c, w0);
                load_k_words<RB>(ktile, t * 16 + 8 + key_r, c, w1);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][n][e] = 0.0f;
#pragma unroll
                for (int k = 0; k < C::KSTEPS; ++k) {
                    uint32_t a[4];
                    k_pairs<KIND>(w0, k, a[0], a[2]);
                    k_pairs<KIND>(w1, k, a[1], a[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(s[t][n], a, qf[k][n][0], qf[k][n][1], kBf16);
                }
            }
            // ---- scale, bias, mask; is a new reference maximum due? ----
            bool raise = false;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float ks = C::kQuant ? sc[t * 16 + g * 8 + key_r] : 1.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) s[t][n][2 * g + e] *= C::kQuant ? factor[n][e] * ks : factor[n][e];
                }
            if (p.is_alibi) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float pos = (float)(key0 + t * 16 + g * 8 + key_r - (con.len - 1));
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) s[t][n][2 * g + e] = fmaf(slope[n][e], pos, s[t][n][2 * g + e]);
                    }
            }
            if (valid != kAllKeys) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const bool masked = !((valid >> (t * 16 + g * 8 + key_r)) & 1u);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) s[t][n][2 * g + e] = masked ? -INFINITY : s[t][n][2 * g + e];
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = s[0][n][e];
#pragma unroll
                    for (int t = 0; t < MT; ++t) top = fmaxf(top, fmaxf(s[t][n][e], s[t][n][2 + e]));
                    raise |= top > m[n][e] + (8.0f + kLift);
                }
            // New units for the weights too, where V rows far larger than those before would leave fp32 in the old ones.
            float v_top = 0.0f;
            if (C::kQuant) {
#pragma unroll
                for (int t = 0; t < MT; ++t) v_top = fmaxf(v_top, fmaxf(sc[TK + t * 16 + key_r], sc[TK + t * 16 + 8 + key_r]));
                raise |= v_top * f_top > power2(kMostScaled);
            }
            if (__any_sync(0xffffffffu, raise)) {
                if (C::kQuant) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, d));
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = m[n][e];
#pragma unroll
                        for (int t = 0; t < MT; ++t) top = fmaxf(top, fmaxf(s[t][n][e], s[t][n][2 + e]) - kLift);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        float shrink = exp2_fast(m[n][e] - top);
                        if (top > m[n][e]) unset |= 1u << (2 * n + e);
                        m[n][e] = top;
                        l[n][e] *= shrink;
                        if (C::kQuant) {
                            const int by = min(0, kMostScaled - exponent(v_top) - exponent(f[n][e]));
                            f[n][e] = __uint_as_float(__float_as_uint(f[n][e]) + ((uint32_t)by << 23));  // times 2^by
                            shrink *= power2(max(-126, by));  // (past that there is nothing to keep)
                        }
#pragma unroll
                        for (int t = 0; t < C::MTILES; ++t) acc[t][n][e] *= shrink, acc[t][n][2 + e] *= shrink;
                    }
                set_f_top();
            }
            // ---- probabilities, weights ----
            bool wide = false;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float vs = C::kQuant ? sc[TK + t * 16 + g * 8 + key_r] : 1.0f;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float pr = exp2_fast(s[t][n][2 * g + e] - m[n][e]);
                            l[n][e] += pr;
                            if (C::kQuant) {
                                s[t][n][2 * g + e] = pr * (vs * f[n][e]);
                                wide |= s[t][n][2 * g + e] > 32768.0f;
                            } else {
                                s[t][n][2 * g + e] = pr;
                            }
                        }
                }
            if (C::kQuant && (__any_sync(0xffffffffu, wide || unset != 0))) {
                // The weights' own reference: the largest of this tile comes to 2^7 if it has outgrown its units, or if it is
                // the first that is not zero since the reference maximum rose (a small weight may then be the one that
                // matters) -- as far as what has been summed up so far still fits fp32.
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = 0.0f;
#pragma unroll
                        for (int t = 0; t < MT; ++t) top = fmaxf(top, fmaxf(s[t][n][e], s[t][n][2 + e]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        float held = 0.0f;
#pragma unroll
                        for (int t = 0; t < C::MTILES; ++t) held = fmaxf(held, fmaxf(fabsf(acc[t][n][e]), fabsf(acc[t][n][2 + e])));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) held = fmaxf(held, __shfl_xor_sync(0xffffffffu, held, d));
                        const int ex = exponent(top);
                        if (ex > -127 && ex < 128 && (ex >= 15 || ((unset >> (2 * n + e)) & 1u))) {
                            unset &= ~(1u << (2 * n + e));
                            // To 2^7 exactly, if nothing is in the way: the weight that matters most is not rounded then.
                            // (by: no less than -102, since a V scale is at most 2^101 in these units, a probability 2^8)
                            const int by = min(min(min(7 - ex, 126), 120 - exponent(f[n][e])), max(0, 100 - exponent(held)));
                            const float g = by == 7 - ex ? 128.0f / top : power2(by);
                            f[n][e] *= g;
#pragma unroll
                            for (int t = 0; t < MT; ++t) s[t][n][e] *= g, s[t][n][2 + e] *= g;
#pragma unroll
                            for (int t = 0; t < C::MTILES; ++t) acc[t][n][e] *= g, acc[t][n][2 + e] *= g;
                        }
                    }
                set_f_top();
            }
            // ---- output ----
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t x;
                        if (kBf16) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(s[t][n][2 * g], s[t][n][2 * g + 1]);
                            x = *reinterpret_cast<const uint32_t *>(&h);
                        } else {
                            const __half2 h = __floats2half2_rn(s[t][n][2 * g], s[t][n][2 * g + 1]);
                            x = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        pf[n][g] = movmatrix(x);
                    }
                uint32_t w[4][C::VW];
#pragma unroll
                for (int j = 0; j < 4; ++j) load_v_words<RB>(vtile, t * 16 + 4 * j + (c ^ (j & 1)), r, w[j]);
#pragma unroll
                for (int x = 0; x < C::VW; ++x) {
                    constexpr int EPW = C::EPW;
                    uint32_t lo[EPW], hi[EPW];
                    v_pairs<KIND>(w[0][x], w[1][x], lo);
                    v_pairs<KIND>(w[2][x], w[3][x], hi);
#pragma unroll
                    for (int e = 0; e < EPW / 2; ++e) {
                        const int tile = x * (EPW / 2) + e;
                        if (tile < C::MTILES) {
                            const uint32_t a[4] = {lo[2 * e], lo[2 * e + 1], hi[2 * e], hi[2 * e + 1]};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma16816(acc[tile][n], a, pf[n][0], pf[n][1], kBf16);
                        }
                    }
                }
            }
        }

        // ---- end of the piece: join the lanes' sums, then the warps that shared its keys ----
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                const float inv = 1.0f / f[n][e];
#pragma unroll
                for (int t = 0; t < C::MTILES; ++t) acc[t][n][e] *= inv, acc[t][n][2 + e] *= inv;
            }
        const int live = (con.end - con.begin + TK - 1) / TK;  // key parts that had a tile, if fewer than there are
        for (int half = p.key_warps / 2; half > 0; half /= 2) {
            if (half >= live) continue;
            const int other = kpart >= half ? kpart - half : kpart;
            float *slot = merge + ((other * p.head_warps + warp % p.head_warps) * NT * 8) * C::kMergeRow;
            if (kpart >= half && kpart < 2 * half) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float *rec = slot + (n * 8 + 2 * c + e) * C::kMergeRow;
#pragma unroll
                        for (int t = 0; t < C::MTILES; ++t) {
                            rec[t * 16 + r] = acc[t][n][e];
                            rec[t * 16 + 8 + r] = acc[t][n][2 + e];
                        }
                        if (r == 0) rec[D] = m[n][e], rec[D + 1] = l[n][e];
                    }
            }
            __syncthreads();
            if (kpart < half) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float *rec = slot + (n * 8 + 2 * c + e) * C::kMergeRow;
                        const float m2 = rec[D], top = fmaxf(m[n][e], m2);
                        const float a = exp2_fast(m[n][e] - top), b = exp2_fast(m2 - top);
                        m[n][e] = top;
                        l[n][e] = l[n][e] * a + rec[D + 1] * b;
#pragma unroll
                        for (int t = 0; t < C::MTILES; ++t) {
                            acc[t][n][e] = acc[t][n][e] * a + rec[t * 16 + r] * b;
                            acc[t][n][2 + e] = acc[t][n][2 + e] * a + rec[t * 16 + 8 + r] * b;
                        }
                    }
            }
            __syncthreads();
        }
        if (kpart == 0 && !idle) {
            const bool whole = con.begin == 0 && con.end == con.len;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int h = n * 8 + 2 * c + e;
                    if (h >= heads) continue;
                    const float inv = l[n][e] > 0.0f ? 1.0f / l[n][e] : (l[n][e] == 0.0f ? 0.0f : l[n][e]);
                    const float lse = l[n][e] == 0.0f ? -INFINITY : (m[n][e] + log2f(l[n][e])) * kLn2;
                    const long long row = (long long)con.b * p.head_q + head0 + h;
                    const long long piece = (span * 2 + (con.begin == 0 ? 1 : 0)) * p.head_q + head0 + h;
                    float *dst32 = whole ? p.own_o + row * D : p.part_o + piece * D;
                    uint16_t *dst16 = static_cast<uint16_t *>(p.o) + (long long)con.b * p.o_row_stride + (long long)(head0 + h) * D;
                    const bool to16 = whole && p.o;
#pragma unroll
                    for (int w = 0; w < C::VW; ++w) {
                        constexpr int kHalfWord = RB & 16;  // the last word has two bytes then
                        const int n_el = kHalfWord && w == C::VW - 1 ? C::EPW / 2 : C::EPW;
                        const int dim = word_offset<RB, 8>(w, r) * C::EPW / 4;
                        float x[C::EPW];
#pragma unroll
                        for (int i = 0; i < C::EPW; ++i) {
                            const int el = w * C::EPW + i;
                            x[i] = el < D / 8 ? acc[el >> 1][n][2 * (el & 1) + e] * inv : 0.0f;
                        }
                        if (to16) {
                            uint32_t y[C::EPW / 2];
#pragma unroll
                            for (int i = 0; i < C::EPW / 2; ++i) {
                                if (p.q_bf16) {
                                    const __nv_bfloat162 z = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                                    y[i] = *reinterpret_cast<const uint32_t *>(&z);
                                } else {
                                    const __half2 z = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                                    y[i] = *reinterpret_cast<const uint32_t *>(&z);
                                }
                            }
                            if (n_el == 8) *reinterpret_cast<uint4 *>(dst16 + dim) = make_uint4(y[0], y[1 % (C::EPW / 2)], y[2 % (C::EPW / 2)], y[3 % (C::EPW / 2)]);
                            else if (n_el == 4) *reinterpret_cast<uint2 *>(dst16 + dim) = make_uint2(y[0], y[1 % (C::EPW / 2)]);
                            else *reinterpret_cast<uint32_t *>(dst16 + dim) = y[0];
                        } else {
#pragma unroll
                            for (int i = 0; i < C::EPW / 2; ++i)
                                if (2 * i < n_el) *reinterpret_cast<float2 *>(dst32 + dim + 2 * i) = make_float2(x[2 * i], x[2 * i + 1]);
                        }
                    }
                    if (r == 0) {
                        if (to16) {
                            if (p.lse) p.lse[row] = lse;
                        } else if (whole) {
                            p.own_lse[row] = lse;
                        } else {
                            p.part_lse[piece] = lse;
                        }
                    }
                }
        }
    }
    if (stays) pdl_wait();
}

template <int KIND, int D, int NT>
cudaError_t launch_stream_variant(const StreamParams &p, cudaStream_t s) {
    using C = StreamCfg<KIND, D, NT>;
    auto kernel = da_stream_kernel<KIND, D, NT>;
    static thread_local uint64_t ready = 0;  // devices on which this thread has raised the kernel's shared-memory limit
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((ready >> dev) & 1u)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    const int streams = p.head_k * p.chunks;
    const dim3 grid(p.spans, (streams + p.head_warps - 1) / p.head_warps);
    count_launch();
    return launch_kernel(kernel, grid, kStreamWarps * 32, C::kSmemBytes, s, true, p);
}

// Query heads of a warp: 16 where the accumulators of two column tiles fit, 8 otherwise.
template <int D>
constexpr int stream_nt(int group) {
    return D <= 128 && group > 8 ? 2 : 1;
}

template <int D>
cudaError_t launch_stream_dim(int kind, bool bf16, const StreamParams &p, cudaStream_t s) {
    if constexpr (D <= 128) {
        if (stream_nt<D>(p.group) == 2) {
            if (kind == 1) return launch_stream_variant<1, D, 2>(p, s);
            if (kind == 2) return launch_stream_variant<2, D, 2>(p, s);
            if (kind == 3) return launch_stream_variant<3, D, 2>(p, s);
            return bf16 ? launch_stream_variant<4, D, 2>(p, s) : launch_stream_variant<0, D, 2>(p, s);
        }
    }
    if (kind == 1) return launch_stream_variant<1, D, 1>(p, s);
    if (kind == 2) return launch_stream_variant<2, D, 1>(p, s);
    if (kind == 3) return launch_stream_variant<3, D, 1>(p, s);
    if constexpr (D <= 128) {
        return bf16 ? launch_stream_variant<4, D, 1>(p, s) : launch_stream_variant<0, D, 1>(p, s);
    }
    return cudaErrorInvalidValue;
}

template <int D>
StreamShape stream_shape_dim(int kind, int group) {
    const int nt = stream_nt<D>(group);
    const int rb = kind == 3 ? D / 2 : (kind ? D : 2 * D);
    return {8 * nt, D <= 128 && nt == 1 && rb <= 128 ? 2 : 1};
}

}  // namespace da
