// Few new tokens over paged KV (paged_varlen.hpp): sequences whose packed rows fit one or two column
// groups of 16 (a single token, drafted tokens, a short turn).
//
// HBM bounds them, so the kernel streams pages as decode does instead of sharing tiles through LDS: a
// workgroup is one (sequence, row tile, KV head, key range), its four waves take the 32-key tiles of the
// range in turn and are merged at the end.
//   S^T[32 keys x 16 NC rows] = K Q^T on v_mfma_f32_16x16x32, K straight from memory in A-operand
//     registers (the head dim permuted alike for K and Q), every K and V fragment used for NC column
//     groups;
//   O^T[D x 16 NC rows] += V^T P^T, V through this wave's own LDS tile and transposed reads.
// 8-bit codes are widened (e4m3.hpp) between memory and the matrix unit. A wave has one tile in flight:
// the next V is requested when V has gone to LDS, the next K behind the QK products.
//
// Measured (MI355X): bf16, 8 sequences of 6 tokens behind 4,096, 32/8 heads, D 128: 30 us, 4.5 TB/s (a
// call 43; through the 128-row kernel of paged_tile.hpp, 24 of its rows in use, 93); fp16, 40 single
// tokens behind 200 to 6,000, D 64: 49 us, 5.2 TB/s; 5 tokens behind 2,300, 8-bit pages: 9.3 us.
#pragma once

#include <hip/hip_runtime.h>

#include "decode_common.hpp"
#include "e4m3.hpp"
#include "paged_varlen.hpp"

namespace sca_hip {
namespace {

typedef uint32_t few_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t few_u32x2 __attribute__((ext_vector_type(2)));

template <int D, bool kHeld8, int NC>
struct FewGeom {
    static constexpr int ROWS = 16 * NC;            // packed rows per unit
    static constexpr int N16 = kHeld8 ? D / 64 : D / 32;  // 16-byte K loads per lane and row
    static constexpr int N8 = kHeld8 ? (D / 32) % 2 : 0;  // and one of 8 bytes
    static constexpr int NK = D / 32;               // QK k steps
    static constexpr int ND = D / 16;               // PV output tiles
    static constexpr int RB = 2 * D;                // bytes of a V row in LDS
    static constexpr int CPR = kHeld8 ? D / 16 : D / 8;   // 16-byte chunks of a row in memory
    static constexpr int NV = kMfmaTile * CPR / kWave;    // V loads per lane and tile
    static constexpr int TILE_BYTES = kMfmaTile * RB;
    static constexpr int V_BYTES = kDecodeWaves * TILE_BYTES;
    // Registers: O and Q of NC groups, a tile's K and V.
    static constexpr int WAVES = FewResident(D, kHeld8, NC);
};

template <typename E>
struct FewMfma;
template <>
struct FewMfma<F16> {
    using M = DecMfma<DecF16>;
};
template <>
struct FewMfma<BF16> {
    using M = DecMfma<DecBF16>;
};

// A unit's work, with LDS for the waves' V tiles and for (m, l).
template <typename E, int D, bool kHeld8, int NC>
__device__ __forceinline__ void FewUnit(const PagedArgs& p, const PagedUnit& u, uint8_t* s_v,
                                        float (*s_m)[16 * NC], float (*s_l)[16 * NC]) {
    using G = FewGeom<D, kHeld8, NC>;
    using M = typename FewMfma<E>::M;
    using vec8 = typename M::vec8;

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16;
    const int grp = lane / 16;

    const PagedSeq& sq = u.seq;
    const int rows = sq.q_count * p.group;
    const int diag = p.causal ? sq.keys - sq.q_count : 0;
    const int visible = VisibleKeys(sq, u.tile, G::ROWS, p.group, p.causal != 0);
    // Key range of this unit, in whole rounds of the four waves.
    constexpr int kRound = kDecodeWaves * kMfmaTile;
    int first = 0, rounds = (visible + kRound - 1) / kRound;
    if (sq.splits > 1) SplitRange((visible + kRound - 1) / kRound, sq.splits, u.split, &first, &rounds);
    const int t_begin = first * kRound;
    const int t_end = min(visible, t_begin + rounds * kRound);

    // Column c * 16 + col of the unit: its packed row, last visible key, query.
    int limit[NC], least = sq.keys - 1;
    vec8 qb[NC][G::NK];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int row = min(u.tile * G::ROWS + 16 * c + col, rows - 1);  // (rows past the last repeat it)
        const int token = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(p.group));
        const int head = u.h_kv * p.group + row - token * p.group;
        limit[c] = p.causal ? min(sq.keys - 1, token + diag) : sq.keys - 1;
        const uint16_t* q_row = static_cast<const uint16_t*>(p.q) +
                                static_cast<int64_t>(sq.q_first + token) * p.q_ss + head * p.q_sh;
#pragma unroll
        for (int j = 0; j < G::NK; ++j) {
            int at = 32 * j + 8 * grp;  // 16-bit pages: k step j of lane group grp
            if constexpr (kHeld8) {
                at = j < 2 * G::N16 ? 64 * (j / 2) + 16 * grp + 8 * (j % 2) : 64 * G::N16 + 8 * grp;
            }
            qb[c][j] = __builtin_bit_cast(vec8, *reinterpret_cast<const uint4*>(q_row + at));
        }
    }
    if (p.causal) {  // the unit's first row sees least
        const int row = min(u.tile * G::ROWS, rows - 1);
        least = min(least, static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(p.group)) + diag);
    }
    const float scale2 = p.scale * kLog2e;

    floatx4 o[NC][G::ND];
    float m[NC], l[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = neg_inf();
        l[c] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < G::ND; ++dt) o[c][dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    constexpr int kEb = kHeld8 ? 1 : 2;
    const uint8_t* k_base = static_cast<const uint8_t*>(p.k) + u.h_kv * p.k_sh * kEb;
    const uint8_t* v_base = static_cast<const uint8_t*>(p.v) + u.h_kv * p.v_sh * kEb;
    const uint32_t k_row = static_cast<uint32_t>(p.k_ss) * kEb, v_row = static_cast<uint32_t>(p.v_ss) * kEb;
    const uint8_t* exp_base = lane < 32 ? p.k_exp : p.v_exp;
    const int32_t* table = p.page_table + static_cast<int64_t>(sq.table_row) * p.max_blocks;
    const uint32_t bs_mask = (1u << p.block_shift) - 1;
    const uint32_t max_blocks = static_cast<uint32_t>(min(p.max_blocks, int64_t{0x7fffffff}));
    const uint32_t num_blocks = static_cast<uint32_t>(p.num_blocks);

    uint8_t* vs = s_v + wave * G::TILE_BYTES;
    const int tr_row = 4 * grp + col / 4;
    const int tr_rd = tr_row * G::RB + 8 * (col % 4);
    const int tr_x = VSwz<D>(tr_row) * 32;

    // Pool row of key lane % 32 of the tile that starts at key t0, or -1 (past the range, unmapped).
    auto row_of = [&](int t0) __attribute__((always_inline)) -> int {
        const uint32_t key = static_cast<uint32_t>(t0) + lane % 32;
        const uint32_t logical = key >> p.block_shift;
        if (key >= static_cast<uint32_t>(t_end) || logical >= max_blocks) return -1;
        const uint32_t id = static_cast<uint32_t>(table[logical]);  // (negative ids are large ones)
        return id < num_blocks ? static_cast<int>((id << p.block_shift) | (key & bs_mask)) : -1;
    };
    few_u32x4 k16[2][G::N16 > 0 ? G::N16 : 1];
    few_u32x2 k8[2];
    few_u32x4 v[G::NV];
    uint32_t next_exponent = 0, next_valid = 0;
    uint32_t k_safe[2];
    auto issue_v = [&](int pool_row) __attribute__((always_inline)) {
        next_valid = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(pool_row >= 0)));
        const uint32_t safe = pool_row < 0 ? 0 : static_cast<uint32_t>(pool_row);
        if constexpr (kHeld8) {
            const uint64_t page_head = static_cast<uint64_t>(safe >> p.block_shift) * static_cast<uint32_t>(p.kv_heads) +
                                       static_cast<uint32_t>(u.h_kv);
            next_exponent = exp_base[(page_head << p.block_shift) + (safe & bs_mask)];
        }
#pragma unroll
        for (int i = 0; i < G::NV; ++i) {
            const int c = i * kWave + lane;
            const uint32_t r = __shfl(safe, c / G::CPR);
            v[i] = *reinterpret_cast<const few_u32x4*>(v_base + static_cast<uint64_t>(r) * v_row + (c % G::CPR) * 16);
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) k_safe[rt] = __shfl(safe, 16 * rt + col);
    };
    auto issue_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const uint8_t* src = k_base + static_cast<uint64_t>(k_safe[rt]) * k_row;
#pragma unroll
            for (int j = 0; j < G::N16; ++j) {
                k16[rt][j] = *reinterpret_cast<const few_u32x4*>(src + 64 * j + 16 * grp);
            }
            if constexpr (G::N8) k8[rt] = *reinterpret_cast<const few_u32x2*>(src + 64 * G::N16 + 8 * grp);
        }
    };
    auto compute = [&](int t0, bool more, int next_row) __attribute__((always_inline)) {
        const uint32_t valid = next_valid, exponent = next_exponent;
        const bool whole = valid == 0xffffffffu;
#pragma unroll
        for (int i = 0; i < G::NV; ++i) {
            const int c = i * kWave + lane;
            const int r = c / G::CPR;
            const int pos = c % G::CPR;
            const uint32_t keep = whole || ((valid >> r) & 1u) ? ~0u : 0u;  // (rows that do not exist may hold a NaN)
            if constexpr (kHeld8) {
                const float unit = UnitOf(__shfl(exponent, 32 + r));
                few_u32x4 lo = __builtin_bit_cast(few_u32x4, Widen8<E>(v[i].x, v[i].y, unit));
                few_u32x4 hi = __builtin_bit_cast(few_u32x4, Widen8<E>(v[i].z, v[i].w, unit));
                if (!whole) lo &= keep, hi &= keep;
                few_u32x4* dst = reinterpret_cast<few_u32x4*>(vs + r * G::RB + ((pos ^ VSwz<D>(r)) * 32));
                dst[0] = lo;
                dst[1] = hi;
            } else {
                few_u32x4 w = v[i];
                if (!whole) w &= keep;
                *reinterpret_cast<few_u32x4*>(vs + r * G::RB + (((pos >> 1) ^ VSwz<D>(r)) * 32) + (pos & 1) * 16) = w;
            }
        }
        if (more) issue_v(next_row);
        floatx4 s[NC][2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const float unit = kHeld8 ? UnitOf(__shfl(exponent, 16 * rt + col)) : 1.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c][rt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            auto step = [&](const vec8& kf, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < NC; ++c) s[c][rt] = M::mma(kf, qb[c][j], s[c][rt]);
            };
#pragma unroll
            for (int j = 0; j < G::N16; ++j) {
                const few_u32x4 w = k16[rt][j];
                if constexpr (kHeld8) {
                    step(__builtin_bit_cast(vec8, Widen8<E>(w.x, w.y, unit)), 2 * j);
                    step(__builtin_bit_cast(vec8, Widen8<E>(w.z, w.w, unit)), 2 * j + 1);
                } else {
                    step(__builtin_bit_cast(vec8, w), j);
                }
            }
            if constexpr (G::N8) {
                step(__builtin_bit_cast(vec8, Widen8<E>(k8[rt].x, k8[rt].y, unit)), G::NK - 1);
            }
        }
        if (more) issue_k();
        const bool masked = !whole || t0 + kMfmaTile - 1 > least;
        vec8 pb[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float sv[2][4];
            float mx = neg_inf();
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = 16 * rt + 4 * grp + i;
                    float x = s[c][rt][i] * scale2;
                    if (masked) x = ((valid >> at) & 1u) && t0 + at <= limit[c] ? x : neg_inf();
                    sv[rt][i] = x;
                    mx = fmaxf(mx, x);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m[c], mx);
            if (__builtin_amdgcn_ballot_w64(m_new > m[c]) != 0) {
                const float alpha = (m[c] == neg_inf()) ? 0.0f : fast_exp2(m[c] - m_new);
                l[c] *= alpha;
#pragma unroll
                for (int dt = 0; dt < G::ND; ++dt) o[c][dt] *= alpha;
                m[c] = m_new;
            }
            const float m_use = (m[c] == neg_inf()) ? 0.0f : m[c];
            // Summed in fp32, rounded once to the 16-bit type for PV; fp16 weights scaled by 2^15 keep all
            // their bits down to 2^-29 (as in decode8.hip).
            float pr[2][4];
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = fast_exp2(sv[rt][i] - m_use);
                    l[c] += w;
                    pr[rt][i] = w * M::kScale;
                }
            }
            pb[c] = __builtin_bit_cast(
                vec8, make_uint4(M::pack(pr[0][0], pr[0][1]), M::pack(pr[0][2], pr[0][3]),
                                 M::pack(pr[1][0], pr[1][1]), M::pack(pr[1][2], pr[1][3])));
        }
        // The tile is this wave's own: its LDS writes and reads stay in order without a barrier.
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
        for (int dt = 0; dt < G::ND; ++dt) {
            const uint8_t* a = vs + tr_rd + ((dt * 32) ^ tr_x);
            const uint2 lo = M::Tr::read(a);
            const uint2 hi = M::Tr::read(a + 16 * G::RB);
            const vec8 vt = __builtin_bit_cast(vec8, make_uint4(lo.x, lo.y, hi.x, hi.y));
#pragma unroll
            for (int c = 0; c < NC; ++c) o[c][dt] = M::mma(vt, pb[c], o[c][dt]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    int t0 = t_begin + wave * kMfmaTile;
    if (t0 < t_end) {
        issue_v(row_of(t0));
        issue_k();
    }
    int row = row_of(t0 + kRound);
    for (; t0 < t_end; t0 += kRound) {
        const int now = row;
        row = row_of(t0 + 2 * kRound);
        compute(t0, t0 + kRound < t_end, now);
    }

    // Merge: the waves' (m, l), then O column group by column group through the V tiles' LDS.
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        if (grp == 0) {
            s_m[wave][16 * c + col] = m[c];
            s_l[wave][16 * c + col] = l[c];
        }
    }
    float* s_o = reinterpret_cast<float*>(s_v);  // [wave][16][D]
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (c > 0) __syncthreads();
#pragma unroll
        for (int dt = 0; dt < G::ND; ++dt) {
            *reinterpret_cast<floatx4*>(s_o + (wave * 16 + col) * D + dt * 16 + 4 * grp) = o[c][dt];
        }
        __syncthreads();
        const int left = min(16, rows - (u.tile * G::ROWS + 16 * c));  // rows of this group (maybe none)
        for (int idx = threadIdx.x; idx < left * (D / 4); idx += kDecodeThreads) {
            const int r = idx / (D / 4);
            const int d = (idx % (D / 4)) * 4;
            float mm = neg_inf();
#pragma unroll
            for (int w = 0; w < kDecodeWaves; ++w) mm = fmaxf(mm, s_m[w][16 * c + r]);
            float lsum = 0.0f;
            floatx4 osum = {0.0f, 0.0f, 0.0f, 0.0f};
            // (also where no wave has a maximum: a NaN among the scores must not become a zero)
#pragma unroll
            for (int w = 0; w < kDecodeWaves; ++w) {
                const float mw = s_m[w][16 * c + r];
                const float wgt = mw == neg_inf() ? 0.0f : fast_exp2(mw - mm);
                lsum += s_l[w][16 * c + r] * wgt;
                osum += *reinterpret_cast<const floatx4*>(s_o + (w * 16 + r) * D + d) * wgt;
            }
            osum *= 1.0f / M::kScale;
            const int packed = u.tile * G::ROWS + 16 * c + r;
            if (sq.splits > 1) {
                const int64_t state =
                    sq.state_base + (static_cast<int64_t>(u.split) * p.kv_heads + u.h_kv) * rows + packed;
                *reinterpret_cast<floatx4*>(p.part_o + state * D + d) = osum;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * state) = make_float2(mm, lsum);
                continue;
            }
            const int token = static_cast<int>(static_cast<uint32_t>(packed) / static_cast<uint32_t>(p.group));
            const int head = u.h_kv * p.group + packed - token * p.group;
            const float inv = lsum > 0.0f ? 1.0f / lsum : lsum;  // (NaN stays NaN)
            const int64_t out_row = static_cast<int64_t>(sq.q_first) + token;
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out_row * p.o_ss + head * p.o_sh + d) =
                make_uint2(M::pack(osum[0] * inv, osum[1] * inv), M::pack(osum[2] * inv, osum[3] * inv));
            if (p.lse != nullptr && d == 0) {
                p.lse[out_row * p.heads + head] = __builtin_bit_cast(uint32_t, lsum) == 0 ? neg_inf() : (mm + __log2f(lsum)) * kLn2;
            }
        }
    }
}

template <typename E, int D, bool kHeld8, int NC>
__global__ __launch_bounds__(kDecodeThreads, (FewGeom<D, kHeld8, NC>::WAVES)) void paged_few_kernel(
    const PagedArgs p, const PagedSeqs seqs) {
    using G = FewGeom<D, kHeld8, NC>;
    __shared__ __align__(16) uint8_t s_v[G::V_BYTES];
    __shared__ float s_m[kDecodeWaves][G::ROWS];
    __shared__ float s_l[kDecodeWaves][G::ROWS];
    FewUnit<E, D, kHeld8, NC>(p, FindUnit(seqs, p.kv_heads, static_cast<int>(blockIdx.x)), s_v, s_m, s_l);
}

}  // namespace

template <typename E, int D, bool kHeld8, int NC>
int LaunchPagedFew(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s) {
    hipLaunchKernelGGL((paged_few_kernel<E, D, kHeld8, NC>), dim3(static_cast<unsigned>(units)),
                       dim3(kDecodeThreads), 0, s, a, seqs);
    return CheckLaunch("paged_few_kernel", s);
}

}  // namespace sca_hip
