// Attention of ragged chunks of new tokens over paged KV: what the kernels and their plan share.
//
// Rows. The query heads of one KV head read the same keys, so their rows share row tiles: packed row
// R of a (sequence, KV head) is new token R / group of head R % group. A chunk of 32 tokens with four
// heads a group is one 128-row tile. Sequences of few rows go to a kernel with tiles of 16 or 32 rows.
// Units. A workgroup takes one unit: (sequence, row tile, key split, KV head). The sequences of a
// launch are listed in the kernel's arguments (PagedSeq), at most kPagedSeqs of them; more go out in
// further launches. So nothing is uploaded, and a captured launch keeps its own list.
// Splits. Where few row tiles meet many keys, a tile's keys are cut into ranges of whole key tiles,
// and every range leaves the unnormalised fp32 state of its rows (O, reference point mu in log2
// units, l) in scratch for paged_combine_kernel.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "flash_common.hpp"
#include "sca_device.hpp"

namespace sca_hip {

constexpr int kPagedRows = 128;   // packed rows per workgroup
constexpr int kPagedSeqs = 112;   // sequences per launch: 32 B each, below 4 KB of arguments

// Workgroups of the few-token kernel that a CU holds: O and Q of its column groups and a tile's K and V
// in registers (as built; more would spill).
constexpr int FewResident(int head_dim, bool held8, int column_groups) {
    const int need = column_groups * (head_dim / 16 * 4 + head_dim / 32 * 4) +
                     (held8 ? head_dim / 4 : head_dim / 2) + 70;
    return need <= 96 ? 5 : need <= 128 ? 4 : need <= 168 ? 3 : need <= 256 ? 2 : 1;
}

// Keys per tile of the general kernel and workgroups of it that a CU holds, by what fits 256 registers a lane.
// Measured (MI355X, us), 64 or 32 keys: 16-bit D 96 145 / 167, D 128 502 / 331 (2 chunks of 1024 tokens behind
// 6,000 to 9,000), 8-bit D 128 (4 of 2048) 1,707 / 1,809; one or two workgroups: D 160 16-bit 421 / 238, 8-bit (5
// of 856 behind 8,535) 1,360 / 810. From D 192 on a workgroup has eight waves.
constexpr int TileKeys(int head_dim, bool held8) {
    return head_dim <= (held8 ? 128 : 96) || head_dim >= 192 ? 64 : 32;
}
constexpr int TileResident(int head_dim) { return head_dim <= 160 ? 2 : 1; }

struct PagedSeq {
    int32_t unit_end;    // units of this and all earlier sequences of the launch
    int32_t q_first;     // first new token's row in q and out
    int32_t q_count;     // new tokens
    int32_t keys;        // keys, the new tokens' included
    int32_t table_row;   // row of the page table
    int32_t splits;      // key splits of its row tiles
    int32_t state_base;  // its first state in scratch (splits > 1)
    int32_t row_tiles;
};

struct PagedSeqs {
    int32_t count;
    int32_t few_units;  // of the few-token kernel, ahead of the others (paged_mixed.hpp)
    PagedSeq seq[kPagedSeqs];
};

struct PagedArgs {
    const void* q;
    const void* k;
    const void* v;
    const uint8_t* k_exp;  // 8-bit pages
    const uint8_t* v_exp;
    void* out;
    float* lse;
    const int32_t* page_table;
    float* part_o;   // [state][D]
    float* part_ml;  // [state][2]
    int64_t max_blocks, num_blocks;
    int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;
    int32_t heads, kv_heads, group, block_shift, causal;
    float scale;
};
static_assert(sizeof(PagedArgs) + sizeof(PagedSeqs) <= 4096, "kernel arguments");

// Launchers, instantiated in the file of their kernel; `units` workgroups.
template <typename E, int D, bool kHeld8>
int LaunchPagedTile(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s);  // paged_tile.hpp
template <typename E, int D>
int LaunchPagedWide(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s);  // paged_wide.hpp
template <typename E, int D>
int LaunchPagedDsplit(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s);  // paged_dsplit.hip
template <typename E, int D>
int LaunchPagedMixed(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s);  // paged_mixed.hpp
template <typename E, int D, bool kHeld8, int NC>
int LaunchPagedFew(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s);  // paged_few.hpp

namespace {

// Unit w of a launch.
struct PagedUnit {
    PagedSeq seq;
    int tile, split, h_kv;
};

__device__ __forceinline__ PagedUnit FindUnit(const PagedSeqs& seqs, int kv_heads, int w) {
    int at = 0;
    if (seqs.count > 1) {
        // Sequences that end at or before unit w: every lane looks at two of them.
        const int lane = threadIdx.x % kWave;
        const int e0 = lane < seqs.count ? seqs.seq[lane].unit_end : 0x7fffffff;
        const int e1 = lane + kWave < seqs.count ? seqs.seq[lane + kWave].unit_end : 0x7fffffff;
        at = __popcll(__builtin_amdgcn_ballot_w64(e0 <= w)) + __popcll(__builtin_amdgcn_ballot_w64(e1 <= w));
        at = __builtin_amdgcn_readfirstlane(at);
    }
    PagedUnit u;
    u.seq = seqs.seq[at];
    const uint32_t local = static_cast<uint32_t>(w - (at > 0 ? seqs.seq[at - 1].unit_end : 0));
    // KV heads fastest: workgroups are dealt to the XCDs in turn, so with 8 KV heads (or a multiple)
    // an XCD's L2 sees the keys of one of them. Longest row tiles first.
    const uint32_t rest = local / static_cast<uint32_t>(kv_heads);
    u.h_kv = static_cast<int>(local - rest * static_cast<uint32_t>(kv_heads));
    const uint32_t t = rest / static_cast<uint32_t>(u.seq.splits);
    u.split = static_cast<int>(rest - t * static_cast<uint32_t>(u.seq.splits));
    u.tile = u.seq.row_tiles - 1 - static_cast<int>(t);
    return u;
}

// Keys that the rows of a tile see at most: all, or up to its last token's own position.
__device__ __forceinline__ int VisibleKeys(const PagedSeq& s, int tile, int tile_rows, int group,
                                           bool causal) {
    if (!causal) return s.keys;
    const int last_row = min((tile + 1) * tile_rows, s.q_count * group) - 1;
    const int last = static_cast<int>(static_cast<uint32_t>(last_row) / static_cast<uint32_t>(group));
    return max(0, min(s.keys, last + s.keys - s.q_count + 1));
}

}  // namespace
}  // namespace sca_hip
