// Long chunks of new tokens over 16-bit pages (paged_varlen.hpp): the wide-row flash kernel
// (flash_wide.hpp, head_dim 32 to 160) with its K and V tiles copied page by page. A wave copies 16
// rows of every 64-key tile, so pages of at least 16 tokens serve it: their ids are uniform per wave,
// come through the scalar cache and cost no vector instruction. The matrix units and the softmax's vector
// work bound it, as they bound the kernel over plain K and V.
//
// Measured (MI355X): bf16, 512 tokens behind 12,289, 32/8 heads, D 128: 126 us with the merge (paged_tile.hpp
// over the same pages 320; K and V without pages 107); 4 chunks of 2048 behind 6,000 to 14,000: 1,657
// us, 968 TF/s; 3 of 300 to 1000 behind 200 to 6,000, D 64: 75 us.
#pragma once

#include <hip/hip_runtime.h>

#include "flash_wide.hpp"
#include "paged_job.hpp"

namespace sca_hip {
namespace {

template <typename E, int D, Denominator kDen>
__global__ __launch_bounds__(WideGeom<D>::THREADS, 1) void paged_wide_kernel(const PagedArgs a,
                                                                             const PagedSeqs seqs) {
    static_assert(WideGeom<D>::BM == kPagedRows);
    sca_flash_params p;
    PagedJob job;
    JobOf(a, FindUnit(seqs, a.kv_heads, static_cast<int>(blockIdx.x)), &p, &job);
    const SplitArgs sp{a.group, 1, a.part_o, a.part_ml};
    const VarlenArgs vl{nullptr, nullptr, nullptr};
    constexpr bool kCausal = true;
    constexpr WideMode kMode = kPaged;
    constexpr int num_q_tiles = 0;
#include "flash_wide_body.hpp"
}

}  // namespace

template <typename E, int D>
int LaunchPagedWide(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s) {
    using G = WideGeom<D>;
    auto launch = [&]<Denominator kDen>() -> int {
        if (const int rc = EnsureLdsLimit<&paged_wide_kernel<E, D, kDen>>(G::LDS_BYTES, "paged LDS limit")) return rc;
        hipLaunchKernelGGL((paged_wide_kernel<E, D, kDen>), dim3(static_cast<unsigned>(units)), dim3(G::THREADS),
                           G::LDS_BYTES, s, a, seqs);
        return CheckLaunch("paged_wide_kernel", s);
    };
    return a.lse != nullptr ? launch.template operator()<DenominatorFor<D>(true)>()
                            : launch.template operator()<DenominatorFor<D>(false)>();
}

}  // namespace sca_hip
