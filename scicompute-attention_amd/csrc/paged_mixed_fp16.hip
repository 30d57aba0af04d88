// The mixed paged kernel's fp16 instantiations.

#include "paged_mixed.hpp"

namespace sca_hip {

template int LaunchPagedMixed<F16, 32>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);
template int LaunchPagedMixed<F16, 64>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);

}  // namespace sca_hip
