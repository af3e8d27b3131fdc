// Launch parameters of the shared-prefix kernel (da_prefix_sm100.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace da {

// How the rows of a KV head -- the `group` query heads of every sequence -- and the tiles of the prefix are dealt out.
// 128-row tiles hold tile_seqs = 128 / group sequences; two row tiles make a unit, which runs over all key tiles.  The
// key tiles of all units, laid end to end, are cut into runs of cta_tiles, one per CTA.
struct PrefixGrid {
    int tile_seqs;   // sequences of a row tile
    int row_tiles;   // row tiles of a KV head
    int pairs;       // units of a KV head: (row_tiles + 1) / 2
    int key_tiles;   // 128-key tiles of the prefix
    int cta_tiles;   // of a CTA; at least, if own_cost is set
    int ctas;
    int max_parts;   // most partial results of a row
    int total;       // key tiles of all units
    // The tensor cores' work on the prefix and the memory's on the sequences' own keys go side by side, each on its SMs:
    // the runs become as long as they have to be for both to end together, and the CTAs without a run leave their SMs to
    // the key stream.  How many own keys there are is known on the device only.
    int own_cost;    // of an own key, in 1/65536 of a key tile's; 0: no sharing
    int sms;
    int most_tiles;             // of a CTA then: the prefix keeps a quarter of the SMs
    unsigned long long by_sms;  // 2^64 / (65536 sms), rounded up
};

// Key tiles of a CTA next to so many own keys (the same in all three kernels of a call, and on the way to their first load:
// no 64-bit division).
__host__ __device__ inline int prefix_run(const PrefixGrid &g, long long keys) {
    const unsigned long long prefix = (unsigned long long)g.total << 16, own = (unsigned long long)keys * (unsigned)g.own_cost;
    if (own < prefix / 8) return g.cta_tiles;  // (not worth the longer runs: 170 us instead of 166 with 9 % of own work)
#ifdef __CUDA_ARCH__
    const long long even = (long long)__umul64hi(prefix + own, g.by_sms);
#else
    const long long even = (long long)(((unsigned __int128)(prefix + own) * g.by_sms) >> 64);
#endif
    // (rounded down: a run's start and end take about a tile longer than a span's)
    return even > g.most_tiles ? g.most_tiles : (even < g.cta_tiles ? g.cta_tiles : (int)even);
}

struct PrefixParams {
    PrefixGrid grid;
    const void *k, *v;                       // [rows, head_k, dim]
    const int *table;                        // optional: pages of the prefix
    long long k_row_stride, v_row_stride;    // in elements
    long long rows;                          // of k and v
    int page_shift;
    int prefix_len;
    int batch, head_q, head_k, group, dim;
    const int *cu_seq_k;                     // lengths of the sequences' own keys
    int is_alibi;
    float scale_log2;
    float *part_o, *part_lse;                // [max_parts][batch][head_q][dim], [max_parts][batch][head_q]
    int *status;
};

// Parts of a row of sequence b and KV head hk: how many, in slots 0 .. n - 1.
__host__ __device__ inline int prefix_parts_of(const PrefixGrid &g, int hk, int b) {
    const int row_tile = b / g.tile_seqs, pair = row_tile / 2;
    const long long unit = (long long)hk * g.pairs + pair;
    const long long first = unit * g.key_tiles / g.cta_tiles, last = ((unit + 1) * g.key_tiles - 1) / g.cta_tiles;
    // A unit of one row tile gives its second stream every other key tile, and each stream leaves a part.
    const int streams = 2 * pair + 1 < g.row_tiles ? 1 : 2;
    return (int)(last - first + 1) * streams;
}

// tm_q: q as [batch][head_q][dim], box {64, group, tile_seqs}; tm_k, tm_v: [rows][head_k][dim], box {64, 1, 128 keys or
// a shorter page}; all with the 128-byte swizzle.
cudaError_t launch_prefix(bool bf16, const PrefixParams &p, const CUtensorMap &tm_q, const CUtensorMap &tm_k,
                          const CUtensorMap &tm_v, cudaStream_t s);

}  // namespace da
