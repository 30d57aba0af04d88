// The paged wide kernel's fp16 instantiations (a file per type, so that they compile in parallel).

#include "paged_wide.hpp"

namespace sca_hip {

#define SCA_INSTANTIATE(D) \
    template int LaunchPagedWide<F16, D>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);
SCA_INSTANTIATE(32)
SCA_INSTANTIATE(64)
SCA_INSTANTIATE(96)
SCA_INSTANTIATE(128)
SCA_INSTANTIATE(160)

}  // namespace sca_hip
