// The streaming decode kernel over e4m3 caches.
#include "sa_stream_kernel.cuh"

namespace sa {

cudaError_t launch_stream_e4m3(const CUtensorMap &mk, const CUtensorMap &mv, const StreamParams &sp, int dtype, int head_dim,
                               int ctas, cudaStream_t stream)
{
    return launch_code<kCodeE4M3>(mk, mv, sp, dtype, head_dim, ctas, stream);
}

}  // namespace sa
