// Key-stream decode kernels (da_stream_kernel.cuh) for head dim 96.
#include "da_stream_kernel.cuh"

namespace da {
cudaError_t launch_stream_d96(int kind, bool bf16, const StreamParams &p, cudaStream_t s) {
    return launch_stream_dim<96>(kind, bf16, p, s);
}
StreamShape stream_shape_d96(int kind, int group) { return stream_shape_dim<96>(kind, group); }
}  // namespace da
