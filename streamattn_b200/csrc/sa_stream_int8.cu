// The streaming decode kernel over int8 caches.
#include "sa_stream_kernel.cuh"

namespace sa {

cudaError_t launch_stream_int8(const CUtensorMap &mk, const CUtensorMap &mv, const StreamParams &sp, int dtype, int head_dim,
                               int ctas, cudaStream_t stream)
{
    return launch_code<kCodeInt8>(mk, mv, sp, dtype, head_dim, ctas, stream);
}

}  // namespace sa
