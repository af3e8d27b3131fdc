// Key-stream decode kernels (da_stream_kernel.cuh) for head dim 64.
#include "da_stream_kernel.cuh"

namespace da {
cudaError_t launch_stream_d64(int kind, bool bf16, const StreamParams &p, cudaStream_t s) {
    return launch_stream_dim<64>(kind, bf16, p, s);
}
StreamShape stream_shape_d64(int kind, int group) { return stream_shape_dim<64>(kind, group); }
}  // namespace da
