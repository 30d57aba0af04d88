// Long chunks of new tokens over 16-bit pages at head_dim 192 and 256: the split-dims flash kernel
// (flash_dsplit.hip) with its K and V tiles copied page by page, as paged_wide.hpp does for the smaller
// head dims. A wave copies 8 rows of every 32-key tile, so pages of 8 tokens will do.
//
// Measured (MI355X): three prompts of 900 to 2600 tokens, 16/4 heads, D 256, LSE: 225 us (paged_tile.hpp)
// -> 115 us. Looking at the page ids of every tile inside the steady loop, instead of once ahead of it
// (FirstHole), takes 8 more scalar registers and another exit from the loop; the compiler then keeps O
// in memory over the loop's head.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "flash_common.hpp"
#include "paged_job.hpp"

namespace sca_hip {
namespace {

template <typename E, int D, Denominator kDen>
__global__ __launch_bounds__(DsplitGeom<D>::THREADS, 1) void paged_dsplit_kernel(const PagedArgs a,
                                                                                 const PagedSeqs seqs) {
    static_assert(DsplitGeom<D>::BM == kPagedRows);
    sca_flash_params p;
    PagedJob job;
    JobOf(a, FindUnit(seqs, a.kv_heads, static_cast<int>(blockIdx.x)), &p, &job);
    const SplitArgs sp{a.group, 1, a.part_o, a.part_ml};
    constexpr bool kCausal = true, kCut = true, kPaged = true;
    constexpr int num_q_tiles = 0;
#include "flash_dsplit_body.hpp"
}

}  // namespace

template <typename E, int D>
int LaunchPagedDsplit(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s) {
    using G = DsplitGeom<D>;
    auto launch = [&]<Denominator kDen>() -> int {
        if (const int rc = EnsureLdsLimit<&paged_dsplit_kernel<E, D, kDen>>(G::LDS_BYTES, "paged LDS limit")) return rc;
        hipLaunchKernelGGL((paged_dsplit_kernel<E, D, kDen>), dim3(static_cast<unsigned>(units)),
                           dim3(G::THREADS), G::LDS_BYTES, s, a, seqs);
        return CheckLaunch("paged_dsplit_kernel", s);
    };
    return a.lse != nullptr ? launch.template operator()<DenominatorFor<D>(true)>()
                            : launch.template operator()<DenominatorFor<D>(false)>();
}

#define SCA_INSTANTIATE(E, D) \
    template int LaunchPagedDsplit<E, D>(const PagedArgs&, const PagedSeqs&, int, hipStream_t);
SCA_INSTANTIATE(F16, 192)
SCA_INSTANTIATE(F16, 256)
SCA_INSTANTIATE(BF16, 192)
SCA_INSTANTIATE(BF16, 256)

}  // namespace sca_hip
