// Long chunks and sequences of up to 16 packed rows in one launch (head_dim 32 and 64, 16-bit pages): the
// wide flash kernel's units, then the few-token kernel's, which fill the CUs that the chunks leave idle.
//
// At these head dims a CU holds two workgroups of the wide kernel (256 registers a lane, 64 KB of LDS), and
// as many of these, enough for the few-token units to stream at HBM's rate. Measured (MI355X), two launches
// -> one: three chunks of 300 to 1000 tokens and 40 single ones behind 200 to 6000, 32/8 heads, D 64: 133.9
// -> 119.9 us; one of 512 and one single, D 64: 49.8 -> 39.4; one of 64 and 100 single, D 64: 116.6 -> 101.9;
// the first at D 32: 92.0 -> 76.8. Few-token units first: 126. From D 96 on a workgroup of the wide kernel
// fills its CU, and so few-token units have half or a third of their waves: D 128, the first case 254 -> 237,
// but one chunk of 100 and 100 single tokens 237 -> 261, one of 512 and 32 single ones 195 -> 205.
#pragma once

#include <hip/hip_runtime.h>

#include "flash_wide.hpp"
#include "paged_few.hpp"
#include "paged_job.hpp"

namespace sca_hip {
namespace {

template <typename E, int D, Denominator kDen>
__global__ __launch_bounds__(WideGeom<D>::THREADS, 1) void paged_mixed_kernel(const PagedArgs a,
                                                                              const PagedSeqs seqs) {
    static_assert(WideGeom<D>::THREADS == kDecodeThreads && WideGeom<D>::BM == kPagedRows);
    // The chunks' units come first, the others fill what they leave.
    const int few = seqs.few_units, wide = static_cast<int>(gridDim.x) - few, at = static_cast<int>(blockIdx.x);
    const int w = at < wide ? few + at : at - wide;
    const PagedUnit u = FindUnit(seqs, a.kv_heads, w);
    if (w < few) {
        using G = FewGeom<D, false, 1>;
        constexpr int kStats = kDecodeWaves * G::ROWS * 4;
        static_assert(G::V_BYTES + 2 * kStats <= WideGeom<D>::LDS_BYTES);
        extern __shared__ __align__(16) uint8_t lds8[];
        FewUnit<E, D, false, 1>(a, u, lds8, reinterpret_cast<float (*)[G::ROWS]>(lds8 + G::V_BYTES),
                                reinterpret_cast<float (*)[G::ROWS]>(lds8 + G::V_BYTES + kStats));
        return;
    }
    sca_flash_params p;
    PagedJob job;
    JobOf(a, u, &p, &job);
    const SplitArgs sp{a.group, 1, a.part_o, a.part_ml};
    const VarlenArgs vl{nullptr, nullptr, nullptr};
    constexpr bool kCausal = true;
    constexpr WideMode kMode = kPaged;
    constexpr int num_q_tiles = 0;
#include "flash_wide_body.hpp"
}

}  // namespace

template <typename E, int D>
int LaunchPagedMixed(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s) {
    using G = WideGeom<D>;
    auto launch = [&]<Denominator kDen>() -> int {
        if (const int rc = EnsureLdsLimit<&paged_mixed_kernel<E, D, kDen>>(G::LDS_BYTES, "paged LDS limit")) return rc;
        hipLaunchKernelGGL((paged_mixed_kernel<E, D, kDen>), dim3(static_cast<unsigned>(units)), dim3(G::THREADS),
                           G::LDS_BYTES, s, a, seqs);
        return CheckLaunch("paged_mixed_kernel", s);
    };
    return a.lse != nullptr ? launch.template operator()<DenominatorFor<D>(true)>()
                            : launch.template operator()<DenominatorFor<D>(false)>();
}

}  // namespace sca_hip
