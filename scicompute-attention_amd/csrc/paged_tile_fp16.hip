// The general paged kernel's fp16 instantiations (a file per type, so that they compile in parallel).

#include "paged_tile.hpp"

namespace sca_hip {

#define SCA_INSTANTIATE(D)                                                                        \
    template int LaunchPagedTile<F16, D, false>(const PagedArgs&, const PagedSeqs&, int, hipStream_t); \
    template int LaunchPagedTile<F16, D, true>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);
SCA_INSTANTIATE(32)
SCA_INSTANTIATE(64)
SCA_INSTANTIATE(96)
SCA_INSTANTIATE(128)
SCA_INSTANTIATE(160)
SCA_INSTANTIATE(192)
SCA_INSTANTIATE(256)

}  // namespace sca_hip
