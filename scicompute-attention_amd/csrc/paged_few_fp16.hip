// The few-token paged kernel's fp16 instantiations (a file per type, so that they compile in parallel).

#include "paged_few.hpp"

namespace sca_hip {

#define SCA_INSTANTIATE(D, NC)                                                                       \
    template int LaunchPagedFew<F16, D, false, NC>(const PagedArgs&, const PagedSeqs&, int, hipStream_t); \
    template int LaunchPagedFew<F16, D, true, NC>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);
SCA_INSTANTIATE(32, 1)
SCA_INSTANTIATE(64, 1)
SCA_INSTANTIATE(96, 1)
SCA_INSTANTIATE(128, 1)
SCA_INSTANTIATE(160, 1)
SCA_INSTANTIATE(192, 1)
SCA_INSTANTIATE(256, 1)
SCA_INSTANTIATE(32, 2)
SCA_INSTANTIATE(64, 2)
SCA_INSTANTIATE(96, 2)
SCA_INSTANTIATE(128, 2)
SCA_INSTANTIATE(160, 2)
SCA_INSTANTIATE(192, 2)

}  // namespace sca_hip
