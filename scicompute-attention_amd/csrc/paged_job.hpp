// A workgroup's unit of a paged launch as the flash kernels take it.
#pragma once

#include <hip/hip_runtime.h>

#include "paged_varlen.hpp"

namespace sca_hip {
namespace {

__device__ __forceinline__ void JobOf(const PagedArgs& a, const PagedUnit& u, sca_flash_params* p, PagedJob* job) {
    const PagedSeq& sq = u.seq;
    *p = sca_flash_params{};
    p->q = a.q, p->k = a.k, p->v = a.v, p->out = a.out, p->lse = a.lse;
    p->batch = 1;
    p->num_heads = a.heads;
    p->num_kv_heads = a.kv_heads;
    p->q_sh = a.q_sh, p->q_ss = a.q_ss;
    p->k_sh = a.k_sh, p->k_ss = a.k_ss;
    p->v_sh = a.v_sh, p->v_ss = a.v_ss;
    p->o_sh = a.o_sh, p->o_ss = a.o_ss;
    p->scale = a.scale;
    // Without a causal mask the diagonal lies behind the last key.
    p->diagonal = a.causal ? sq.keys - sq.q_count : sq.keys;
    *job = PagedJob{};
    job->table = a.page_table + static_cast<int64_t>(sq.table_row) * a.max_blocks;
    job->max_blocks = a.max_blocks, job->num_blocks = a.num_blocks;
    job->block_shift = a.block_shift;
    job->q_first = sq.q_first, job->q_count = sq.q_count, job->keys = sq.keys;
    job->tile = u.tile, job->split = u.split, job->splits = sq.splits, job->h_kv = u.h_kv;
    job->state = sq.state_base + (static_cast<int64_t>(u.split) * a.kv_heads + u.h_kv) * sq.q_count * a.group;
}

}  // namespace
}  // namespace sca_hip
