// The general kernel of attention over paged KV (paged_varlen.hpp): 8-bit pages, pages of fewer than 16
// tokens (8 from head_dim 192 on), and rows of pages more than 2^25 elements apart. The matrix units bound it.
//
// Four waves of 32 packed rows; key tiles of 64 or 32 keys (TileKeys) come through registers into two LDS
// buffers: while a tile is multiplied the next one's loads are in flight, and 8-bit codes are widened
// (e4m3.hpp) on their way into LDS, once per workgroup, so that one inner loop serves both kinds of pages.
// A lane looks up the page of one key per tile, one tile ahead of the loads that need it, and hands the row to
// the lanes that copy it with a shuffle. Formulation, swizzles and online softmax are those of the flash
// kernels (flash_common.hpp). Two waves to a SIMD, so that one's vector work runs beside the other's products:
// two workgroups to a CU where the registers allow (TileResident); from head_dim 192 on O and Q of 32 rows leave
// no room, and eight waves work in pairs instead. A pair's waves score 32 keys of a tile each, agree on the
// row maxima and swap their weights through LDS, and each multiplies all of them into half of the dims.
//
// Measured (MI355X): 4 chunks of 2048 tokens behind 6,000 to 14,000, 8-bit pages, 32/8 heads, D 128: 1,707
// us (940 TF/s; the wide kernel over 16-bit pages of the same lengths 1,657). Vector instructions per MFMA
// decide: 8.3 now, 10.3 before pool rows were multiplied in 32 bits, whole tiles left unmasked and maxima
// taken without regard to NaN (1,880 us). A higher wave priority over the products changes nothing. Pairs, against
// four waves with all dims: D 192 8-bit pages (3 chunks of 1,295 to 3,885 tokens) 586 -> 444, 16-bit (2 of 1024)
// 814 -> 548; D 256 8-bit (2 of 1024, 16/4 heads) 549 -> 460.
#pragma once

#include <hip/hip_runtime.h>

#include "e4m3.hpp"
#include "paged_varlen.hpp"

namespace sca_hip {
namespace {

template <int D, bool kHeld8>
struct TileGeom {
    static constexpr bool PAIRS = D >= 192;            // two waves share 32 rows
    static constexpr int THREADS = PAIRS ? 512 : 256;
    static constexpr int BN = TileKeys(D, kHeld8);     // keys per tile
    static constexpr int NT = BN / 32;                 // S^T tiles of 32 keys
    static constexpr int KS = D / 16;
    static constexpr int DT = D / 32 / (PAIRS ? 2 : 1);  // O^T tiles of a wave
    static constexpr int RB = 2 * D;                   // LDS row bytes
    static constexpr int TILE_BYTES = BN * RB;
    static constexpr int CPR = kHeld8 ? D / 16 : D / 8;  // 16-byte chunks of a row in memory
    static constexpr int CHUNKS = BN * CPR;
    static constexpr int PER = (CHUNKS + THREADS - 1) / THREADS;  // chunks per thread
    // Two buffers of K and V; pairs: their weights ([wave][k step][lane], 16 bytes) and maxima ([wave][row]).
    static constexpr int P_BASE = 4 * TILE_BYTES;
    static constexpr int MAX_BASE = P_BASE + (PAIRS ? THREADS * 32 : 0);
    static constexpr int LDS_BYTES = MAX_BASE + (PAIRS ? THREADS * 2 : 0);
    // First dim of chunk c (8 dims) of an LDS row. 8-bit pages: a lane widens 16 codes to the chunks p and
    // p + CPR, so that the lanes of a row write neighbouring chunks (as 2p and 2p + 1 they collide in the
    // banks: 1,724 instead of 1,707 us at the size above, D 256 570 instead of 556). Q's dims are permuted
    // as K's are, and those of V go back to their places with the output.
    static constexpr __device__ int ChunkDim(int c) { return !kHeld8 ? 8 * c : c < CPR ? 16 * c : 16 * (c - CPR) + 8; }
    static_assert(CHUNKS % kWave == 0, "a wave copies a chunk on all lanes or on none (shuffles)");
    static constexpr int WAVES = TileResident(D) * THREADS / 256;  // per SIMD
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));  // (a plain vector stays in registers)

// log2 headroom of the weights: they are 2^(x - mu) with mu that much below the row's maximum. fp16
// weights then keep all their bits down to 2^-21 of the largest (2^-14 without), and stay finite: at
// most 2^(7 + kRescaleSlack).
template <typename E>
struct WeightBias {
    static constexpr float value = 0.0f;
};
template <>
struct WeightBias<F16> {
    static constexpr float value = 7.0f;
};

template <typename E, int D, bool kHeld8>
__global__ __launch_bounds__((TileGeom<D, kHeld8>::THREADS), (TileGeom<D, kHeld8>::WAVES)) void paged_tile_kernel(
    const PagedArgs p, const PagedSeqs seqs) {
    using G = TileGeom<D, kHeld8>;
    using M = Mfma<E>;
    using vec8 = typename E::vec8;
    constexpr int BN = G::BN;
    constexpr float kBias = WeightBias<E>::value;

    extern __shared__ __align__(16) uint8_t lds8[];
    uint8_t* lds_k = lds8;
    uint8_t* lds_v = lds8 + 2 * G::TILE_BYTES;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int lane = tid % kWave;
    const int lr = lane & 31;
    const int hh = lane >> 5;

    const PagedUnit u = FindUnit(seqs, p.kv_heads, static_cast<int>(blockIdx.x));
    const PagedSeq& sq = u.seq;
    const int rows = sq.q_count * p.group;
    const int diag = p.causal ? sq.keys - sq.q_count : 0;
    const int visible = VisibleKeys(sq, u.tile, kPagedRows, p.group, p.causal != 0);
    const int all_tiles = (visible + BN - 1) / BN;
    int first = 0, n_tiles = all_tiles;
    if (sq.splits > 1) SplitRange(all_tiles, sq.splits, u.split, &first, &n_tiles);

    // This lane's row, its token and head; rows past the last one repeat it and are not stored.
    const int rg = wave % 4, part = wave / 4;  // pairs: keys 32 part .. of a tile, dims part * D/2 .. of O
    const int row = u.tile * kPagedRows + 32 * rg + lr;
    const bool row_ok = row < rows;
    const int safe_row = min(row, rows - 1);
    const int token = static_cast<int>(static_cast<uint32_t>(safe_row) / static_cast<uint32_t>(p.group));
    const int head = u.h_kv * p.group + safe_row - token * p.group;
    const int limit = p.causal ? min(sq.keys - 1, token + diag) : sq.keys - 1;  // last visible key
    // The wave's least limit: tiles that end at or before it need no mask for it.
    const int wave_row = min(u.tile * kPagedRows + 32 * rg, rows - 1);
    const int wave_limit =
        p.causal ? min(sq.keys - 1, static_cast<int>(static_cast<uint32_t>(wave_row) /
                                                     static_cast<uint32_t>(p.group)) + diag)
                 : sq.keys - 1;

    vec8 qf[G::KS];
    {
        const uint16_t* q_row = static_cast<const uint16_t*>(p.q) +
                                static_cast<int64_t>(sq.q_first + token) * p.q_ss + head * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) {
            qf[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const uint4*>(q_row + G::ChunkDim(2 * ks + hh)));
        }
    }

    constexpr int kEb = kHeld8 ? 1 : 2;
    const uint8_t* k_base = static_cast<const uint8_t*>(p.k) + u.h_kv * p.k_sh * kEb;
    const uint8_t* v_base = static_cast<const uint8_t*>(p.v) + u.h_kv * p.v_sh * kEb;
    const uint32_t k_row_bytes = static_cast<uint32_t>(p.k_ss) * kEb, v_row_bytes = static_cast<uint32_t>(p.v_ss) * kEb;
    const int32_t* table = p.page_table + static_cast<int64_t>(sq.table_row) * p.max_blocks;
    const uint32_t bs_mask = (1u << p.block_shift) - 1;
    const uint32_t max_blocks = static_cast<uint32_t>(min(p.max_blocks, int64_t{0x7fffffff}));
    const uint32_t num_blocks = static_cast<uint32_t>(p.num_blocks);
    const int end = min(sq.keys, (first + n_tiles) * BN);

    // Pool row of key lane % BN of tile t, or -1 (past the keys, unmapped, outside the pool).
    auto row_of = [&](int t) __attribute__((always_inline)) -> int {
        const int key = t * BN + lane % BN;
        const uint32_t logical = static_cast<uint32_t>(key) >> p.block_shift;
        if (key >= end || logical >= max_blocks) return -1;
        const uint32_t id = static_cast<uint32_t>(table[logical]);  // (negative ids are large ones)
        return id < num_blocks ? static_cast<int>((id << p.block_shift) | (static_cast<uint32_t>(key) & bs_mask)) : -1;
    };
    u32x4 kr[G::PER], vr[G::PER];
    uint32_t k_byte = 0, v_byte = 0;  // exponent bytes of key lane % BN
    uint64_t valid = 0;               // keys of the tile in flight that exist (bit per key)
    auto issue = [&](int pool_row) __attribute__((always_inline)) {
        valid = __builtin_amdgcn_ballot_w64(pool_row >= 0);
        const int safe = pool_row < 0 ? 0 : pool_row;
        if constexpr (kHeld8) {
            const uint32_t at_row = static_cast<uint32_t>(safe);
            const uint64_t at = ((static_cast<uint64_t>(at_row >> p.block_shift) * static_cast<uint32_t>(p.kv_heads) +
                                  static_cast<uint32_t>(u.h_kv)) << p.block_shift) + (at_row & bs_mask);
            k_byte = p.k_exp[at];
            v_byte = p.v_exp[at];
        }
#pragma unroll
        for (int i = 0; i < G::PER; ++i) {
            const int c = i * G::THREADS + tid;
            if (G::CHUNKS % G::THREADS != 0 && c >= G::CHUNKS) continue;
            const uint64_t r = static_cast<uint32_t>(__shfl(safe, c / G::CPR));
            kr[i] = *reinterpret_cast<const u32x4*>(k_base + r * k_row_bytes + (c % G::CPR) * 16);
            vr[i] = *reinterpret_cast<const u32x4*>(v_base + r * v_row_bytes + (c % G::CPR) * 16);
        }
    };
    // Registers -> LDS buffer `buf`. V rows of keys that do not exist are cleared: their weights are
    // zero, but the row may hold a NaN.
    auto Widen = [](uint32_t lo, uint32_t hi, float unit) __attribute__((always_inline)) {
        return __builtin_bit_cast(u32x4, Widen8<E>(lo, hi, unit));
    };
    auto put = [&](int buf) __attribute__((always_inline)) {
        uint8_t* dk = lds_k + buf * G::TILE_BYTES;
        uint8_t* dv = lds_v + buf * G::TILE_BYTES;
        const bool whole = valid == ~uint64_t{0};
#pragma unroll
        for (int i = 0; i < G::PER; ++i) {
            const int c = i * G::THREADS + tid;
            if (G::CHUNKS % G::THREADS != 0 && c >= G::CHUNKS) continue;
            const int r = c / G::CPR;
            const int pos = c % G::CPR;
            uint32_t keep = (valid >> r) & 1 ? ~0u : 0u;
            if constexpr (kHeld8) {
                const float ku = UnitOf(__shfl(k_byte, r)), vu = UnitOf(__shfl(v_byte, r));
                const u32x4 k0 = Widen(kr[i].x, kr[i].y, ku), k1 = Widen(kr[i].z, kr[i].w, ku);
                u32x4 v0 = Widen(vr[i].x, vr[i].y, vu), v1 = Widen(vr[i].z, vr[i].w, vu);
                if (!whole) {
                    asm volatile("" : "+v"(keep));  // (a branch: as selects these are a tenth of the step's VALU work)
                    v0 &= keep, v1 &= keep;
                }
                *reinterpret_cast<u32x4*>(dk + r * G::RB + ((pos ^ SwzK<D>(r)) * 16)) = k0;
                *reinterpret_cast<u32x4*>(dk + r * G::RB + (((pos + G::CPR) ^ SwzK<D>(r)) * 16)) = k1;
                *reinterpret_cast<u32x4*>(dv + r * G::RB + ((pos ^ SwzV<D>(r)) * 16)) = v0;
                *reinterpret_cast<u32x4*>(dv + r * G::RB + (((pos + G::CPR) ^ SwzV<D>(r)) * 16)) = v1;
            } else {
                *reinterpret_cast<u32x4*>(dk + r * G::RB + ((pos ^ SwzK<D>(r)) * 16)) = kr[i];
                *reinterpret_cast<u32x4*>(dv + r * G::RB + ((pos ^ SwzV<D>(r)) * 16)) = whole ? vr[i] : vr[i] & keep;
            }
        }
    };

    floatx16 o[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
    }
    float mu = neg_inf();  // reference point of the weights (log2 units)
    float l = 0.0f;        // this lane's share of the denominator
    const float scale2 = p.scale * kLog2e;

    // Fragment positions (flash_common.hpp).
    const int grp = lane >> 4;
    const int sl = lane & 15;
    const int v_key = 4 * hh + (sl >> 2);
    const int v_chunk = 2 * (grp & 1) + ((sl & 3) >> 1);
    const int v_half = (sl & 1) * 8;
    const int dt0 = part * G::DT;  // this wave's first O^T tile

    auto compute = [&](int buf, int t, uint64_t keys_ok) __attribute__((always_inline)) {
        const uint8_t* sk = lds_k + buf * G::TILE_BYTES;
        const uint8_t* sv = lds_v + buf * G::TILE_BYTES;
        constexpr int NT = G::PAIRS ? 1 : G::NT;  // S^T tiles of this wave, from key 32 * n0 on
        const int n0 = G::PAIRS ? part : 0;
        floatx16 s[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int kr_ = 32 * (n + n0) + lr;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                const uint4 f = *reinterpret_cast<const uint4*>(sk + kr_ * G::RB +
                                                                (((2 * ks + hh) ^ SwzK<D>(kr_)) * 16));
                s[n] = M::mma(__builtin_bit_cast(vec8, f), qf[ks], s[n]);
            }
        }
        if (keys_ok != ~uint64_t{0} || t * BN + BN - 1 > wave_limit) {
            const int base = t * BN + 4 * hh;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int k_in = 32 * (n + n0) + 8 * (i / 4) + (i % 4);
                    const bool seen = base + k_in <= limit && ((keys_ok >> (k_in + 4 * hh)) & 1);
                    s[n][i] = seen ? s[n][i] : neg_inf();
                }
            }
        }
        float mx = Max16(s[0]);
        if constexpr (NT > 1) mx = fmaxf(mx, Max16(s[NT - 1]));
        mx = HalfMax(mx);
        if constexpr (G::PAIRS) {
            // The row's maximum over both waves' keys, so that both move their reference point alike.
            float* all = reinterpret_cast<float*>(lds8 + G::MAX_BASE);
            if (hh == 0) all[wave * 32 + lr] = mx;
            __syncthreads();
            mx = fmaxf(mx, all[(wave ^ 4) * 32 + lr]);
        }
        const float top = mx * scale2;
        if (__builtin_amdgcn_ballot_w64(top > mu + kBias + kRescaleSlack) != 0) {
            const bool grow = top > mu + kBias + kRescaleSlack;
            const float mu_new = grow ? top - kBias : mu;
            const float alpha = grow ? fast_exp2(mu - mu_new) : 1.0f;  // 0 where mu was -inf
            mu = mu_new;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt) o[dt] *= alpha;
        }
        const float neg_mu = mu == neg_inf() ? 0.0f : -mu;
        vec8 pb[2 * G::NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = fast_exp2(fmaf(s[n][2 * i], scale2, neg_mu));
                const float b = fast_exp2(fmaf(s[n][2 * i + 1], scale2, neg_mu));
                l += a + b;
                // Rounded once to the 16-bit type, by at most half a step, as the output is.
                w[i] = M::pack(a, b);
            }
            pb[2 * n] = __builtin_bit_cast(vec8, make_uint4(w[0], w[1], w[2], w[3]));
            pb[2 * n + 1] = __builtin_bit_cast(vec8, make_uint4(w[4], w[5], w[6], w[7]));
        }
        if constexpr (G::PAIRS) {
            // Own weights in pb[0, 1], the partner's in pb[2, 3].
            u32x4* all = reinterpret_cast<u32x4*>(lds8 + G::P_BASE) + lane;
#pragma unroll
            for (int i = 0; i < 2; ++i) all[(2 * wave + i) * kWave] = __builtin_bit_cast(u32x4, pb[i]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) pb[2 + i] = __builtin_bit_cast(vec8, all[(2 * (wave ^ 4) + i) * kWave]);
        }
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt) {
#pragma unroll
            for (int n = 0; n < G::NT; ++n) {
                const int keys_of = G::PAIRS ? n ^ part : n;  // (the S^T tile that pb[2 n] is of)
                const uint8_t* a = sv + (32 * keys_of + v_key) * G::RB +
                                   (((4 * (dt + dt0) + v_chunk) ^ SwzV<D>(v_key)) * 16) + v_half;
#pragma unroll
                for (int ps = 0; ps < 2; ++ps) {
                    const uint2 lo = TrRead<E>::read(a + (16 * ps) * G::RB);
                    const uint2 hi = TrRead<E>::read(a + (16 * ps + 8) * G::RB);
                    o[dt] = M::mma(__builtin_bit_cast(vec8, make_uint4(lo.x, lo.y, hi.x, hi.y)),
                                   pb[2 * n + ps], o[dt]);
                }
            }
        }
    };

    if (n_tiles > 0) {
        issue(row_of(first));
        int next = row_of(first + 1);
        put(0);
        uint64_t now_ok = valid;
        __syncthreads();
        for (int j = 0; j < n_tiles; ++j) {
            const bool more = j + 1 < n_tiles;
            if (more) {
                issue(next);
                next = row_of(first + j + 2);
            }
            compute(j & 1, first + j, now_ok);
            if (more) {
                put((j + 1) & 1);
                now_ok = valid;
            }
            __syncthreads();
        }
    }

    float l_all = HalfSum(l);
    if constexpr (G::PAIRS) {
        float* all = reinterpret_cast<float*>(lds8 + G::MAX_BASE);  // (behind the last tile's barrier)
        if (hh == 0) all[wave * 32 + lr] = l_all;
        __syncthreads();
        l_all += all[(wave ^ 4) * 32 + lr];
    }
    const bool first_part = part == 0;
    if (sq.splits > 1) {
        const int64_t state = sq.state_base + (static_cast<int64_t>(u.split) * p.kv_heads + u.h_kv) * rows + row;
        if (row_ok && hh == 0 && first_part) *reinterpret_cast<float2*>(p.part_ml + 2 * state) = make_float2(mu, l_all);
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt) {
            float a[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) a[i] = o[dt][i];
            StorePartialTile(p.part_o + state * D, hh, row_ok, a, [&](int c) { return G::ChunkDim(4 * (dt + dt0) + c); });
        }
        return;
    }
    const float inv = l_all > 0.0f ? 1.0f / l_all : l_all;  // (NaN stays NaN)
    uint16_t* out_row = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(sq.q_first + token) * p.o_ss +
                        head * p.o_sh;
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt) {
        float a[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) a[i] = o[dt][i] * inv;
        StoreTile<M>(out_row, hh, row_ok, a, [&](int c) { return G::ChunkDim(4 * (dt + dt0) + c); });
    }
    if (p.lse != nullptr && row_ok && hh == 0 && first_part) {
        p.lse[static_cast<int64_t>(sq.q_first + token) * p.heads + head] =
            __builtin_bit_cast(uint32_t, l_all) == 0 ? neg_inf() : (mu + __log2f(l_all)) * kLn2;
    }
}

}  // namespace

template <typename E, int D, bool kHeld8>
int LaunchPagedTile(const PagedArgs& a, const PagedSeqs& seqs, int units, hipStream_t s) {
    using G = TileGeom<D, kHeld8>;
    if (const int rc = EnsureLdsLimit<&paged_tile_kernel<E, D, kHeld8>>(G::LDS_BYTES, "paged LDS limit")) return rc;
    hipLaunchKernelGGL((paged_tile_kernel<E, D, kHeld8>), dim3(static_cast<unsigned>(units)), dim3(G::THREADS),
                       G::LDS_BYTES, s, a, seqs);
    return CheckLaunch("paged_tile_kernel", s);
}

}  // namespace sca_hip
