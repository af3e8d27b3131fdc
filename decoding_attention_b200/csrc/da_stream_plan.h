// Host side of the key-stream kernels, shared by the entry points that launch them (da_cache_api.cu).
#pragma once

#include <cstddef>

#include "da_stream.h"

namespace da {

int failf(int code, const char *fmt, ...);  // records the message (da_last_error), returns `code`
int sm_count(int *out);                     // of the current device
bool head_dim_supported(int64_t dim);
bool quantised_kind(int32_t kv_dtype);
// Fills chunks, head_warps, key_warps, spans and min_span from head_k and group.
void plan_stream(int dim, int kind, int sms, StreamParams *p);
size_t stream_piece_bytes(const StreamParams &p, int dim);  // of part_o and part_lse together
int run_stream(int dim, int kind, bool bf16, const StreamParams &p, cudaStream_t s);

}  // namespace da
