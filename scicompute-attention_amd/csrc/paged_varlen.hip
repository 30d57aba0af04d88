// Attention of ragged chunks of new tokens over paged KV: the plan of a call (units, key splits, the
// launches' sequence lists), the merge of key splits, the checks and the C entry points. The kernels are in
// paged_wide.hpp, paged_dsplit.hip, paged_tile.hpp, paged_few.hpp and paged_mixed.hpp; paged_varlen.hpp
// describes rows, units and splits.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <map>
#include <string>
#include <vector>

#include "paged_varlen.hpp"

namespace sca_hip {
namespace {

constexpr int kCombineThreads = 256;
constexpr int64_t kMostScratch = int64_t{64} << 20;

// out = sum_s O_s 2^(mu_s - mu*) / sum_s l_s 2^(mu_s - mu*), one thread per (row, 4 dims); grid.y is
// the sequence. A range that saw no key left zeros.
template <typename E>
__global__ __launch_bounds__(kCombineThreads) void paged_combine_kernel(const PagedArgs p,
                                                                        const PagedSeqs seqs,
                                                                        uint32_t head_dim) {
    using M = Mfma<E>;
    const PagedSeq sq = seqs.seq[blockIdx.y];
    if (sq.splits <= 1) return;
    const uint32_t rows = static_cast<uint32_t>(sq.q_count) * static_cast<uint32_t>(p.group);
    const uint32_t all = rows * static_cast<uint32_t>(p.kv_heads);
    const uint32_t quads = head_dim / 4;
    const uint32_t idx = blockIdx.x * kCombineThreads + threadIdx.x;
    const uint32_t at = idx / quads;  // (KV head, packed row)
    if (at >= all) return;
    const uint32_t d0 = (idx - at * quads) * 4;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + sq.state_base + at;
    const float* po = p.part_o + (static_cast<int64_t>(sq.state_base) + at) * head_dim + d0;
    // Up to sixteen states at a time, all requested before the first is used, so that a merge waits for
    // memory once or twice: with four at a time, twice over for the maximum, 18 states of 160 rows took
    // 12.8 us (6.2 so).
    float mu = neg_inf();
    float l = 0.0f;
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto merge = [&]<int kAtOnce>(int s0) __attribute__((always_inline)) {
        float2 st[kAtOnce];
        floatx4 v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int64_t s = min(s0 + i, sq.splits - 1);  // (repeats of the last one do not count)
            st[i] = ml[s * all];
            v[i] = *reinterpret_cast<const floatx4*>(po + s * all * head_dim);
        }
        float top = mu;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, st[i].x);
        const float back = mu == neg_inf() ? 1.0f : fast_exp2(mu - top);
        l *= back;
#pragma unroll
        for (int d = 0; d < 4; ++d) a[d] *= back;
        mu = top;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            // (a state without a maximum is zeros, or NaN where its scores were, which must stay)
            const float w = st[i].x == neg_inf() ? 1.0f : fast_exp2(st[i].x - mu);
            if (s0 + i < sq.splits) {
                l = fmaf(st[i].y, w, l);
#pragma unroll
                for (int d = 0; d < 4; ++d) a[d] = fmaf(v[i][d], w, a[d]);
            }
        }
    };
    if (sq.splits == 2) {
        merge.template operator()<2>(0);
    } else if (sq.splits <= 4) {
        merge.template operator()<4>(0);
    } else {
        for (int s0 = 0; s0 < sq.splits; s0 += 16) merge.template operator()<16>(s0);
    }
    const float inv = l > 0.0f ? 1.0f / l : l;
    const uint32_t h_kv = at / rows;
    const uint32_t row = at - h_kv * rows;
    const uint32_t token = row / static_cast<uint32_t>(p.group);
    const int64_t head = h_kv * p.group + (row - token * p.group);
    const int64_t out_row = static_cast<int64_t>(sq.q_first) + token;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out_row * p.o_ss + head * p.o_sh + d0) =
        make_uint2(M::pack(a[0] * inv, a[1] * inv), M::pack(a[2] * inv, a[3] * inv));
    if (p.lse != nullptr && d0 == 0) {
        p.lse[out_row * p.heads + head] = l == 0.0f ? neg_inf() : (mu + __log2f(l)) * kLn2;
    }
}

bool Aligned(const void* ptr, uintptr_t bytes) {
    return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0;
}

// The kernels that serve a call: tiles of 128 rows (the flash kernels over pages, or the general one), or
// the few-token kernel's 16 or 32.
enum Kind { kFlash, kTile, kFew16, kFew32, kMixed };

struct Launch {
    Kind kind;
    PagedSeqs seqs;
    int64_t units;
    int64_t combine_rows;  // most (KV head, row) pairs of a split sequence; 0: no merge
    int64_t states;        // that it leaves
};

struct Plan {
    std::vector<Launch> launches;
    int64_t states = 0;  // most states a launch leaves
};

// Sequences of up to 32 packed rows take the few-token kernel (16 at head_dim 256, where two column
// groups of O do not fit the registers): 8 of 24 rows over 4,102 keys took 93 us a call through tiles of 128
// rows, 46 through its 32 (as both kernels were then).
Kind KindFor(const sca_paged_varlen_params& p, int64_t rows) {
    if (rows <= 16) return kFew16;
    if (rows <= 32) return p.head_dim <= 192 ? kFew32 : kFew16;
    // (the flash kernels copy 16 or 8 rows of a page at a time, and address them with 32-bit offsets)
    const bool flash = p.k_exp == nullptr && p.block_size >= (p.head_dim <= 160 ? 16 : 8) && p.k_ss < (1 << 25) &&
                       p.v_ss < (1 << 25);
    return flash ? kFlash : kTile;
}

bool IsFew(Kind kind) { return kind == kFew16 || kind == kFew32; }
int RowsPerTile(Kind kind) { return !IsFew(kind) ? kPagedRows : kind == kFew32 ? 32 : 16; }

// Keys that a workgroup takes in one step.
int KeysPerStep(Kind kind, const sca_paged_varlen_params& p) {
    const int d = static_cast<int>(p.head_dim);
    return IsFew(kind) ? 128 : kind == kTile ? TileKeys(d, p.k_exp != nullptr) : d <= 160 ? 64 : 32;
}

// Workgroups that the GPU holds at once.
int64_t Resident(Kind kind, const sca_paged_varlen_params& p) {
    const int d = static_cast<int>(p.head_dim);
    const int on_cu = kind == kFlash   ? (d <= 64 ? 2 : 1)
                      : kind == kTile ? TileResident(d)
                                      : FewResident(d, p.k_exp != nullptr, kind == kFew32 ? 2 : 1);
    return static_cast<int64_t>(CuCount()) * on_cu;
}

struct Entry {
    PagedSeq seq;
    int64_t steps;   // of its last row tile
    int64_t steps0;  // of its first (the same without a causal mask)
};

// Splits that keep a unit to `span` steps, where that saves enough of them to be worth the states'
// traffic.
int32_t SplitsFor(Kind kind, int64_t steps, int64_t span) {
    if (steps - span < (IsFew(kind) ? 3 : 8)) return 1;
    return static_cast<int32_t>(std::min<int64_t>(64, (steps + span - 1) / span));
}

// Longest units first.
void Order(std::vector<Entry>* list) {
    std::stable_sort(list->begin(), list->end(), [](const Entry& a, const Entry& b) {
        return a.steps * b.seq.splits > b.steps * a.seq.splits;
    });
}

// Steps (about a microsecond each) until the last of the units ends, each given to the workgroup slot that
// is free first; a sequence's row tiles in up to four groups of equal length. What a unit does besides its
// steps counts as `overhead` of them, the merge as `merge` and the states' way through memory.
// Measured (MI355X, us), planned / every unit with all its keys: 512 tokens behind 12,289, D 128 141 / 202; 8 of
// 6 behind 4,096 37.6 / 77.2; 5 behind 2,300, 8-bit pages 18.6 / 39.0; 3 chunks and 40 single tokens, D 64 115 /
// 138. Where the rows fill the GPU it splits nothing (1,000 tokens behind 3,000).
constexpr size_t kSimulated = 32;
int64_t Makespan(const std::vector<Entry>& list, const sca_paged_varlen_params& p, Kind kind, int64_t resident) {
    const int64_t overhead = IsFew(kind) ? 2 : 6, merge = 5;
    std::map<int64_t, int64_t> free_at;  // slots by the time they are free
    free_at[0] = resident;
    int64_t end = 0, states = 0;
    for (const Entry& e : list) {
        const int64_t groups = std::min<int64_t>(4, e.seq.row_tiles);
        for (int64_t g = groups - 1; g >= 0; --g) {
            const int64_t steps = e.steps0 + (e.steps - e.steps0) * (2 * g + 1) / (2 * groups);
            int64_t units = (e.seq.row_tiles * (g + 1) / groups - e.seq.row_tiles * g / groups) * e.seq.splits *
                            p.num_kv_heads;
            const int64_t takes = (steps + e.seq.splits - 1) / e.seq.splits + overhead;
            if (units > 16 * resident) {  // many rounds alike
                const int64_t rounds = units / resident - 8;
                std::map<int64_t, int64_t> later;
                for (const auto& slot : free_at) later[slot.first + rounds * takes] = slot.second;
                free_at.swap(later);
                units -= rounds * resident;
            }
            while (units > 0) {
                const auto first = free_at.begin();
                const int64_t time = first->first, n = std::min(units, first->second);
                if (n == first->second) {
                    free_at.erase(first);
                } else {
                    first->second -= n;
                }
                free_at[time + takes] += n;
                end = std::max(end, time + takes);
                units -= n;
            }
        }
        if (e.seq.splits > 1) states += static_cast<int64_t>(e.seq.q_count) * p.num_heads * e.seq.splits;
    }
    return states == 0 ? end : end + merge + states * (p.head_dim + 2) / 500000;
}

// The launches of one kind, appended to `plan`. States of split keys may go to `most_states` of scratch.
void PlanKind(const sca_paged_varlen_params& p, Kind kind, int64_t most_states, Plan* plan) {
    const int64_t group = p.num_heads / p.num_kv_heads;
    const int64_t rows_per_tile = RowsPerTile(kind);
    const int64_t keys = KeysPerStep(kind, p);
    std::vector<Entry> list;
    int64_t work = 0;  // steps of all units
    for (int64_t s = 0; s < p.num_seqs; ++s) {
        const int64_t n = p.cu_seqlens_q[s + 1] - p.cu_seqlens_q[s];
        if (n == 0 || KindFor(p, n * group) != kind) continue;
        Entry e{};
        e.seq.q_first = p.cu_seqlens_q[s];
        e.seq.q_count = static_cast<int32_t>(n);
        e.seq.keys = p.kv_lens[s];
        e.seq.table_row = p.table_rows != nullptr ? p.table_rows[s] : static_cast<int32_t>(s);
        e.seq.splits = 1;
        e.seq.row_tiles = static_cast<int32_t>((n * group + rows_per_tile - 1) / rows_per_tile);
        e.steps = (p.kv_lens[s] + keys - 1) / keys;
        const int64_t seen = p.kv_lens[s] - n + std::min<int64_t>(n, (rows_per_tile + group - 1) / group);
        e.steps0 = p.causal ? std::max<int64_t>(0, (seen + keys - 1) / keys) : e.steps;
        work += p.num_kv_heads * e.seq.row_tiles * ((e.steps + e.steps0 + 1) / 2);
        list.push_back(e);
    }
    if (list.empty()) return;
    const int64_t resident = Resident(kind, p);
    if (most_states > 0) {
        const int64_t share = std::max<int64_t>(1, (work + resident - 1) / resident);
        int64_t span = share;
        if (list.size() <= kSimulated) {
            // The span of keys per unit with the least estimated run, from half a workgroup's share of
            // the work to all keys.
            int64_t least = -1;
            for (const int quarters : {2, 3, 4, 5, 6, 8, 12, 1 << 20}) {
                const int64_t tried = std::max<int64_t>(IsFew(kind) ? 1 : 4, share * quarters / 4);
                for (Entry& e : list) e.seq.splits = SplitsFor(kind, e.steps, tried);
                Order(&list);
                const int64_t run = Makespan(list, p, kind, resident);
                if (least < 0 || run < least) {
                    least = run;
                    span = tried;
                }
            }
        }
        for (Entry& e : list) e.seq.splits = SplitsFor(kind, e.steps, span);
    }
    Order(&list);
    for (size_t at = 0; at < list.size(); at += kPagedSeqs) {
        Launch launch{};
        launch.kind = kind;
        int64_t states = 0;
        for (size_t i = at; i < std::min(list.size(), at + kPagedSeqs); ++i) {
            PagedSeq q = list[i].seq;
            const int64_t rows = q.q_count * group * p.num_kv_heads;
            while (q.splits > 1 && states + rows * q.splits > most_states) --q.splits;
            q.state_base = static_cast<int32_t>(states);
            if (q.splits > 1) {
                states += rows * q.splits;
                launch.combine_rows = std::max(launch.combine_rows, rows);
            }
            launch.units += static_cast<int64_t>(q.row_tiles) * q.splits * p.num_kv_heads;
            q.unit_end = static_cast<int32_t>(launch.units);  // (Validate bounds the units)
            launch.seqs.seq[launch.seqs.count++] = q;
        }
        launch.states = states;
        plan->states = std::max(plan->states, states);
        plan->launches.push_back(launch);
    }
}

// Joins a launch of long chunks and one of single tokens (paged_mixed.hpp).
void Mix(int64_t most_states, Plan* plan) {
    auto& all = plan->launches;
    auto is = [](Kind kind) { return [kind](const Launch& l) { return l.kind == kind; }; };
    const auto flash = std::find_if(all.begin(), all.end(), is(kFlash));
    const auto few = std::find_if(all.begin(), all.end(), is(kFew16));
    if (flash == all.end() || few == all.end()) return;
    const int64_t states = flash->states + few->states;
    if (flash->seqs.count + few->seqs.count > kPagedSeqs || states > most_states) return;
    Launch both = *few;
    both.kind = kMixed;
    both.seqs.few_units = static_cast<int32_t>(few->units);
    for (int i = 0; i < flash->seqs.count; ++i) {
        PagedSeq q = flash->seqs.seq[i];
        q.unit_end += both.seqs.few_units;
        q.state_base += static_cast<int32_t>(few->states);
        both.seqs.seq[both.seqs.count++] = q;
    }
    both.units += flash->units;
    both.states = states;
    both.combine_rows = std::max(both.combine_rows, flash->combine_rows);
    plan->states = std::max(plan->states, states);
    *flash = both;
    all.erase(few);
}

// Long chunks first: the few-token launches fill the GPU behind them.
Plan MakePlan(const sca_paged_varlen_params& p, int64_t most_states) {
    Plan plan;
    for (Kind kind : {kFlash, kTile, kFew32, kFew16}) PlanKind(p, kind, most_states, &plan);
    if (p.head_dim <= 64) Mix(most_states, &plan);
    return plan;
}

int64_t StateBytes(int64_t head_dim) { return 4 * (head_dim + 2); }

template <typename E, int D, bool kHeld8>
int LaunchKind(const PagedArgs& a, const Launch& l, hipStream_t s) {
    const int units = static_cast<int>(l.units);
    if (l.kind == kTile) return LaunchPagedTile<E, D, kHeld8>(a, l.seqs, units, s);
    if constexpr (!kHeld8) {
        if constexpr (D <= 64) {
            if (l.kind == kMixed) return LaunchPagedMixed<E, D>(a, l.seqs, units, s);
        }
        if (l.kind == kFlash) {
            if constexpr (D <= 160) return LaunchPagedWide<E, D>(a, l.seqs, units, s);
            else return LaunchPagedDsplit<E, D>(a, l.seqs, units, s);
        }
    }
    if constexpr (D <= 192) {
        if (l.kind == kFew32) return LaunchPagedFew<E, D, kHeld8, 2>(a, l.seqs, units, s);
    }
    return LaunchPagedFew<E, D, kHeld8, 1>(a, l.seqs, units, s);
}

template <typename E>
int LaunchOne(const PagedArgs& a, const Launch& l, int64_t head_dim, hipStream_t s) {
    const bool held8 = a.k_exp != nullptr;
    switch (head_dim) {
#define SCA_CASE(D) \
    case D: return held8 ? LaunchKind<E, D, true>(a, l, s) : LaunchKind<E, D, false>(a, l, s);
        SCA_CASE(32)
        SCA_CASE(64)
        SCA_CASE(96)
        SCA_CASE(128)
        SCA_CASE(160)
        SCA_CASE(192)
        SCA_CASE(256)
#undef SCA_CASE
        default: break;
    }
    return SetError(SCA_E_UNSUPPORTED_HEAD_DIM,
                    "paged varlen: head_dim=" + std::to_string(head_dim) + " is not instantiated");
}

template <typename E>
int Run(const sca_paged_varlen_params& p, const Plan& plan, void* scratch, hipStream_t s) {
    PagedArgs a{};
    a.q = p.q, a.k = p.k, a.v = p.v, a.k_exp = p.k_exp, a.v_exp = p.v_exp;
    a.out = p.out, a.lse = p.lse, a.page_table = p.page_table;
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = a.part_o + plan.states * p.head_dim;
    a.max_blocks = p.max_blocks_per_seq, a.num_blocks = p.num_kv_blocks;
    a.q_ss = p.q_ss, a.q_sh = p.q_sh, a.k_ss = p.k_ss, a.k_sh = p.k_sh;
    a.v_ss = p.v_ss, a.v_sh = p.v_sh, a.o_ss = p.o_ss, a.o_sh = p.o_sh;
    a.heads = static_cast<int32_t>(p.num_heads);
    a.kv_heads = static_cast<int32_t>(p.num_kv_heads);
    a.group = static_cast<int32_t>(p.num_heads / p.num_kv_heads);
    while ((int64_t{1} << a.block_shift) < p.block_size) ++a.block_shift;
    a.causal = p.causal;
    a.scale = p.scale;
    for (const Launch& l : plan.launches) {
        int rc = LaunchOne<E>(a, l, p.head_dim, s);
        if (rc != 0) return rc;
        if (l.combine_rows == 0) continue;
        const int64_t threads = l.combine_rows * (p.head_dim / 4);
        const dim3 grid(static_cast<unsigned>((threads + kCombineThreads - 1) / kCombineThreads),
                        static_cast<unsigned>(l.seqs.count));
        hipLaunchKernelGGL((paged_combine_kernel<E>), grid, dim3(kCombineThreads), 0, s, a, l.seqs,
                           static_cast<uint32_t>(p.head_dim));
        rc = CheckLaunch("paged_combine_kernel", s);
        if (rc != 0) return rc;
    }
    return 0;
}

// Everything that can be checked without the pointers' targets; `pointers` false leaves those out.
int Validate(const sca_paged_varlen_params* p, bool pointers) {
    auto fail = [](int code, const std::string& what) { return SetError(code, "paged varlen: " + what); };
    if (p == nullptr) return fail(SCA_E_SHAPE_MISMATCH, "null params");
    if (p->cu_seqlens_q == nullptr || p->kv_lens == nullptr) {
        return fail(SCA_E_SHAPE_MISMATCH, "null cu_seqlens_q or kv_lens (host arrays)");
    }
    if (pointers) {
        if (p->q == nullptr || p->k == nullptr || p->v == nullptr || p->out == nullptr ||
            p->page_table == nullptr) {
            return fail(SCA_E_SHAPE_MISMATCH, "null pointer");
        }
        if ((p->k_exp == nullptr) != (p->v_exp == nullptr)) {
            return fail(SCA_E_SHAPE_MISMATCH, "k_exp and v_exp must both be set (8-bit pages) or both NULL");
        }
        if (!Aligned(p->q, 16) || !Aligned(p->k, 16) || !Aligned(p->v, 16) || !Aligned(p->out, 16)) {
            return fail(SCA_E_LAYOUT_MISMATCH, "q, k, v and out must be 16 B aligned");
        }
    }
    if (p->num_seqs < 1 || p->num_seqs > 0x7fffffffLL / 2) {
        return fail(SCA_E_SHAPE_MISMATCH, "num_seqs=" + std::to_string(p->num_seqs));
    }
    if (p->num_heads < 1 || p->num_heads > 65535 || p->num_kv_heads < 1 || p->num_heads % p->num_kv_heads != 0) {
        return fail(SCA_E_SHAPE_MISMATCH, "invalid heads (H_q=" + std::to_string(p->num_heads) +
                                              ", H_kv=" + std::to_string(p->num_kv_heads) + ")");
    }
    if (p->head_dim % 32 != 0 || p->head_dim < 32 || p->head_dim > 256 || p->head_dim == 224) {
        return fail(SCA_E_UNSUPPORTED_HEAD_DIM, "head_dim=" + std::to_string(p->head_dim));
    }
    if (p->dtype != SCA_DTYPE_F16 && p->dtype != SCA_DTYPE_BF16) {
        return fail(SCA_E_UNSUPPORTED_DTYPE, "computes in fp16/bf16; dtype id " + std::to_string(p->dtype));
    }
    if (!(p->scale > 0.0f) || p->scale > 3.0e38f) {
        return fail(SCA_E_SHAPE_MISMATCH, "scale must be positive and finite");
    }
    const int64_t bs = p->block_size;
    if (bs < 1 || (bs & (bs - 1)) != 0 || p->max_blocks_per_seq < 1 || p->num_kv_blocks < 1 ||
        p->num_kv_blocks > 0x7fffffffLL / bs) {
        return fail(SCA_E_SHAPE_MISMATCH,
                    "block_size must be a power of two, max_blocks_per_seq and num_kv_blocks positive, and the "
                    "pool's tokens below 2^31");
    }
    const bool held8 = p->k_exp != nullptr;
    if (held8 && bs < 8) return fail(SCA_E_SHAPE_MISMATCH, "8-bit pages hold at least 8 tokens");
    const int64_t ve = held8 ? 16 : 8;
    if (p->q_ss % 8 || p->q_sh % 8 || p->o_ss % 8 || p->o_sh % 8 || p->k_ss % ve || p->k_sh % ve ||
        p->v_ss % ve || p->v_sh % ve) {
        return fail(SCA_E_LAYOUT_MISMATCH, "strides must be multiples of 16 B");
    }
    if (p->k_ss < 0 || p->k_ss >= (1LL << 30) || p->v_ss < 0 || p->v_ss >= (1LL << 30)) {
        return fail(SCA_E_LAYOUT_MISMATCH, "K and V row strides must be below 2^30 and not negative");
    }
    const int64_t group = p->num_heads / p->num_kv_heads;
    int64_t units = 0;
    if (p->cu_seqlens_q[0] < 0) return fail(SCA_E_SHAPE_MISMATCH, "cu_seqlens_q starts below 0");
    for (int64_t s = 0; s < p->num_seqs; ++s) {
        const int64_t n = static_cast<int64_t>(p->cu_seqlens_q[s + 1]) - p->cu_seqlens_q[s];
        if (n < 0) {
            return fail(SCA_E_SHAPE_MISMATCH, "cu_seqlens_q decreases at sequence " + std::to_string(s));
        }
        if (p->kv_lens[s] < 0) {
            return fail(SCA_E_SHAPE_MISMATCH, "kv_lens[" + std::to_string(s) + "]=" + std::to_string(p->kv_lens[s]));
        }
        if (p->table_rows != nullptr && p->table_rows[s] < 0) {
            return fail(SCA_E_SHAPE_MISMATCH, "table_rows[" + std::to_string(s) + "] is negative");
        }
        // Keys, and a sequence's rows over its KV heads, are 32-bit numbers in the kernels (with room
        // for a tile past the end).
        if (p->kv_lens[s] > 0x7fffffff - 4096 || n > 0x7fffffffLL / (p->num_heads * (p->head_dim / 4)) - kPagedRows) {
            return fail(SCA_E_SEQ_TOO_LONG, "sequence " + std::to_string(s) + " of " + std::to_string(n) +
                                                " new tokens and " + std::to_string(p->kv_lens[s]) + " keys");
        }
        units += (n * group + 15) / 16 * p->num_kv_heads;  // (no kernel has fewer rows to a unit)
    }
    if (units > 0x7fffffffLL / 64) {
        return fail(SCA_E_SEQ_TOO_LONG, "grid of " + std::to_string(units) + " row tiles exceeds the launch limit");
    }
    return 0;
}

}  // namespace
}  // namespace sca_hip

using sca_hip::SetError;

extern "C" {

int64_t sca_hip_paged_varlen_bytes(const sca_paged_varlen_params* params) {
    if (sca_hip::Validate(params, /*pointers=*/false) != 0) return 0;
    try {
        const int64_t state = sca_hip::StateBytes(params->head_dim);
        return sca_hip::MakePlan(*params, sca_hip::kMostScratch / state).states * state;
    } catch (const std::exception&) {  // no host memory for the plan: the run will say so
        return 0;
    }
}

int sca_hip_paged_varlen(const sca_paged_varlen_params* params, void* scratch, int64_t scratch_bytes,
                         void* stream) {
    if (const int rc = sca_hip::Validate(params, /*pointers=*/true)) return rc;
    if (!sca_hip::Aligned(scratch, 16)) {
        return SetError(SCA_E_LAYOUT_MISMATCH, "paged varlen: scratch must be 16 B aligned");
    }
    const int64_t state = sca_hip::StateBytes(params->head_dim);
    const int64_t room = scratch != nullptr && scratch_bytes > 0
                             ? std::min(scratch_bytes, sca_hip::kMostScratch) / state
                             : 0;
    try {
        const sca_hip::Plan plan = sca_hip::MakePlan(*params, room);
        hipStream_t s = static_cast<hipStream_t>(stream);
        return params->dtype == SCA_DTYPE_F16 ? sca_hip::Run<sca_hip::F16>(*params, plan, scratch, s)
                                              : sca_hip::Run<sca_hip::BF16>(*params, plan, scratch, s);
    } catch (const std::exception& e) {
        return SetError(SCA_E_WORKSPACE, std::string("paged varlen: no host memory for the plan: ") + e.what());
    }
}

}  // extern "C"
