// Long chunks of new tokens over 16-bit pages (paged_varlen.hpp): the wide-row flash kernel
// (flash_wide.hpp, head_dim 32 to 160) with its K and V tiles copied page by page. A wave copies 16
// rows of every 64-key tile, so pages of at least 16 tokens serve it: their ids are uniform per wave,
// come through the scalar cache and cost no vector instruction.
#pragma once

#include <hip/hip_runtime.h>

#include "flash_wide.hpp"
#include "paged_varlen.hpp"

namespace sca_hip {
namespace {

template <typename E, int D, Denominator kDen>
__global__ __launch_bounds__(WideGeom<D>::THREADS, 1) void paged_wide_kernel(const PagedArgs a,
                                                                             const PagedSeqs seqs) {
    static_assert(WideGeom<D>::BM == kPagedRows);
    const PagedUnit u = FindUnit(seqs, a.kv_heads);
    const PagedSeq& sq = u.seq;
    sca_flash_params p{};
    p.q = a.q, p.k = a.k, p.v = a.v, p.out = a.out, p.lse = a.lse;
    p.batch = 1;
    p.num_heads = a.heads;
    p.num_kv_heads = a.kv_heads;
    p.q_sh = a.q_sh, p.q_ss = a.q_ss;
    p.k_sh = a.k_sh, p.k_ss = a.k_ss;
    p.v_sh = a.v_sh, p.v_ss = a.v_ss;
    p.o_sh = a.o_sh, p.o_ss = a.o_ss;
    p.scale = a.scale;
    // Without a causal mask the diagonal lies behind the last key.
    p.diagonal = a.causal ? sq.keys - sq.q_count : sq.keys;
    PagedJob job{};
    job.table = a.page_table + static_cast<int64_t>(sq.table_row) * a.max_blocks;
    job.max_blocks = a.max_blocks, job.num_blocks = a.num_blocks;
    job.block_shift = a.block_shift;
    job.q_first = sq.q_first, job.q_count = sq.q_count, job.keys = sq.keys;
    job.tile = u.tile, job.split = u.split, job.splits = sq.splits, job.h_kv = u.h_kv;
    job.state = sq.state_base + (static_cast<int64_t>(u.split) * a.kv_heads + u.h_kv) * sq.q_count * a.group;
    FlashWide<E, D, true, kPaged, kDen>(p, 0, VarlenArgs{nullptr, nullptr, nullptr},
                                        SplitArgs{a.group, 1, a.part_o, a.part_ml}, job);
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
