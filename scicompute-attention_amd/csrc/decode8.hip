// Decode (one query token per sequence) over pages that keep K and V in 8 bits (e4m3.hpp), and the
// checks of its entry point. Semantics, partial-state layout, split ranges, longest-first schedule and
// combine are those of the 16-bit decode (decode.hip); K and V are the values the codes stand for.
//
// HBM bounds it: D + 1 bytes per key, KV head and tensor, half of what 16-bit pages cost, so that a
// wave has half the time for a tile. The kernel computes as the 16-bit MFMA kernel does (S^T = K Q^T
// with the query heads of a GQA group as the 16 columns, O^T += V^T P^T, 32 tokens a tile) and widens
// the codes on the way:
//   * K: 16 codes of a token row per lane load, widened in registers to the fragments of two k steps
//     (the head dim is permuted alike for K and Q). The row's exponent is the conversion's own scale
//     operand, so scores need no further factor.
//   * V: a lane takes 16 codes of a row, widens them (exponent included) and writes them to this
//     wave's LDS tile in 16 bits; the transposed reads then find what the 16-bit kernel's DMA leaves.
//     V stands in the tile as the 16-bit numbers it stands for, so that P needs no factor per token
//     (in fp16 a weight times a small 2^k would leave the type's range).
//   * Exponents: one byte load per lane and tile (lanes 0-31 the tokens of K, 32-63 of V), handed to
//     the lanes that need them with shuffles.
//
// Measured (MI355X): bf16, 64 sequences of 512 to 16,384 tokens, 32/8 heads, D 128: 194 us, 5.35 TB/s; 16 of
// 3,000 to 5,200, D 96: 24.3 us (4.4); fp16, 1 x 1500, D 128: 6.5 us, a start, six tiles and a merge.

#include <hip/hip_runtime.h>

#include <string>

#include "decode_common.hpp"
#include "decode_order.hpp"
#include "e4m3.hpp"
#include "sca_device.hpp"

namespace sca_hip {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int D>
struct Dec8Geom {
    static constexpr int N16 = D / 64;            // 16-byte K loads per lane and row
    static constexpr int N8 = (D / 32) % 2;       // and one of 8 bytes where D / 32 is odd
    static constexpr int NK = D / 32;             // QK k steps
    static constexpr int ND = D / 16;             // PV output tiles
    static constexpr int RB = 2 * D;              // bytes of a widened V row
    static constexpr int CPR = D / 16;            // 16-code chunks per row
    static constexpr int NV = kMfmaTile * CPR / kWave;  // V loads per lane and tile
    static constexpr int TILE_BYTES = kMfmaTile * RB;
    // Waves per SIMD that the registers are kept to (O, Q and a tile's codes); more than one also keeps
    // O in the ordinary registers, where its rescaling needs no copies.
    static constexpr int WAVES = D <= 32 ? 6 : D <= 64 ? 5 : D <= 96 ? 4 : D <= 128 ? 3 : 2;
    static_assert(NV * kWave == kMfmaTile * CPR, "V chunks divide evenly");
    static_assert(kDecodeWaves * kMfmaHeads * D * 4 <= kDecodeWaves * TILE_BYTES, "merge fits the tiles");
};

template <typename E, int D, bool kWaveHeads>
__global__ __launch_bounds__(kDecodeThreads, Dec8Geom<D>::WAVES) void decode8_kernel(
    const sca_decode_params p, const uint8_t* __restrict__ k_exp, const uint8_t* __restrict__ v_exp,
    int h_chunks, int block_shift) {
    using G = Dec8Geom<D>;
    using T = typename E::Type;
    using M = DecMfma<typename E::Dec>;
    using vec8 = typename M::vec8;

    __shared__ __align__(16) uint8_t s_v[kDecodeWaves * G::TILE_BYTES];
    __shared__ int32_t s_rank[kRankBatch];
    __shared__ int32_t s_seq[2];
    __shared__ float s_m[kDecodeWaves][kMfmaHeads];
    __shared__ float s_l[kDecodeWaves][kMfmaHeads];

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16;
    const int grp = lane / 16;

    const int64_t split = blockIdx.x;
    const int64_t slots = p.num_kv_heads * h_chunks;
    const int64_t hh = kWaveHeads ? static_cast<int64_t>(blockIdx.y) * kDecodeWaves + wave
                                  : static_cast<int64_t>(blockIdx.y);
    const bool slot_ok = hh < slots;
    const uint32_t slot = slot_ok ? static_cast<uint32_t>(hh) : 0;
    const int64_t h_kv = slot / static_cast<uint32_t>(h_chunks);
    const int64_t h_chunk = slot % static_cast<uint32_t>(h_chunks);
    // The sequence of this workgroup: the blockIdx.z-th longest, as in the 16-bit kernel.
    int64_t b = blockIdx.z;
    int len = static_cast<int>(p.seq_kv);  // (below 2^31, as every token index here)
    if (p.seq_lens != nullptr && p.batch <= kRankBatch) {
        const int tid = threadIdx.x;
        const int nb = static_cast<int>(p.batch);
        if (tid < nb) s_rank[tid] = p.seq_lens[tid];
        __syncthreads();
        if (tid < nb) {
            const int mine = s_rank[tid];
            int rank = 0;
            for (int j = 0; j < nb; ++j) {
                const int other = s_rank[j];
                rank += (other > mine) | ((other == mine) & (j < tid));
            }
            if (rank == static_cast<int>(blockIdx.z)) {
                s_seq[0] = tid;
                s_seq[1] = mine;
            }
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(s_seq[0]);
        len = __builtin_amdgcn_readfirstlane(s_seq[1]);
    } else if (p.batch_order != nullptr) {
        const int2 e = reinterpret_cast<const int2*>(p.batch_order)[blockIdx.z];
        b = e.x;
        len = e.y;
    } else if (p.seq_lens != nullptr) {
        len = p.seq_lens[b];
    }
    const int64_t group = static_cast<uint32_t>(p.num_heads) / static_cast<uint32_t>(p.num_kv_heads);
    const int64_t h0 = h_kv * group + h_chunk * kMfmaHeads;
    const int hc = static_cast<int>(group - h_chunk * kMfmaHeads < kMfmaHeads
                                        ? group - h_chunk * kMfmaHeads
                                        : kMfmaHeads);
    const float scale2 = p.scale * kLog2e;

    // Q^T B operand, permuted as K is: k steps 2j and 2j + 1 hold elements 64j + 16 grp .. + 16, the
    // last one of an odd number 8 elements from 64 N16 + 8 grp.
    vec8 qb[G::NK];
    {
        const uint16_t* q_row = static_cast<const uint16_t*>(p.q) + b * p.q_sb + (h0 + col) * p.q_sh;
#pragma unroll
        for (int j = 0; j < G::NK; ++j) {
            const int at = j < 2 * G::N16 ? 64 * (j / 2) + 16 * grp + 8 * (j % 2) : 64 * G::N16 + 8 * grp;
            const uint4 raw = col < hc ? *reinterpret_cast<const uint4*>(q_row + at) : make_uint4(0, 0, 0, 0);
            qb[j] = __builtin_bit_cast(vec8, raw);
        }
    }

    floatx4 o[G::ND];
#pragma unroll
    for (int dt = 0; dt < G::ND; ++dt) o[dt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = neg_inf();  // running max of head `col` (log2 units, identical across lane groups)
    float l = 0.0f;       // this lane's share of the running denominator

    const int chunk = static_cast<int>(SplitChunk(len, p.num_splits));
    const int t_begin = static_cast<int>(min(static_cast<int64_t>(len), split * chunk));
    const int t_end = len - t_begin < chunk ? len : t_begin + chunk;
    const int n_tiles =
        slot_ok && t_end > t_begin ? static_cast<int>((static_cast<uint32_t>(t_end - t_begin) + kMfmaTile - 1) / kMfmaTile)
                                   : 0;
    constexpr int TS = kWaveHeads ? 1 : kDecodeWaves;  // tile stride of one wave

    const uint8_t* k_base = static_cast<const uint8_t*>(p.k) + h_kv * p.k_sh;
    const uint8_t* v_base = static_cast<const uint8_t*>(p.v) + h_kv * p.v_sh;
    const uint8_t* exp_base = lane < 32 ? k_exp : v_exp;
    const int32_t* table = p.page_table + b * p.max_blocks_per_seq;
    const uint32_t bs_mask = (1u << block_shift) - 1;
    // Pool rows and row strides are below 2^31 (checked): one 32 x 32 -> 64 bit product per address.
    const uint32_t k_row = static_cast<uint32_t>(p.k_ss), v_row = static_cast<uint32_t>(p.v_ss);
    const uint32_t max_blocks = static_cast<uint32_t>(min(p.max_blocks_per_seq, int64_t{0x7fffffff}));
    const uint32_t num_blocks = static_cast<uint32_t>(p.num_kv_blocks);

    uint8_t* vs = s_v + wave * G::TILE_BYTES;
    const int tr_row = 4 * grp + col / 4;
    const int tr_rd = tr_row * G::RB + 8 * (col % 4);
    const int tr_x = VSwz<D>(tr_row) * 32;

    // Row of token lane % 32 of a tile (< 0: it contributes nothing). Fetched a tile ahead of the
    // tile's loads, which need it.
    auto row_of = [&](int tile) -> int {
        const uint32_t tok = static_cast<uint32_t>(t_begin) + static_cast<uint32_t>(tile) * kMfmaTile + lane % 32;
        const uint32_t logical = tok >> block_shift;
        if (tok >= static_cast<uint32_t>(t_end) || logical >= max_blocks) return -1;
        const uint32_t id = static_cast<uint32_t>(table[logical]);  // (negative ids are large ones)
        return id < num_blocks ? static_cast<int>((id << block_shift) | (tok & bs_mask)) : -1;
    };
    // A tile's codes on their way, in registers: V is widened into LDS first, and the next tile's V
    // requested into the same registers at once; K likewise behind the QK products. (Two sets of
    // registers halve the waves that fit: measured slower.)
    u32x4 k16[2][G::N16 > 0 ? G::N16 : 1];
    u32x2 k8[2];
    u32x4 v[G::NV];
    uint32_t next_exponent = 0;  // of token lane % 32: K's in the lower half of the wave, V's in the upper
    uint32_t next_valid = 0;     // tokens that exist
    uint32_t k_safe[2];          // rows of this lane's two K rows
    auto issue_v = [&](int row) __attribute__((always_inline)) {
        next_valid = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(row >= 0)));
        const uint32_t safe = row < 0 ? 0 : static_cast<uint32_t>(row);  // rows that count for nothing read row 0
        const uint64_t page_head = static_cast<uint64_t>(safe >> block_shift) * static_cast<uint32_t>(p.num_kv_heads) +
                                   static_cast<uint32_t>(h_kv);
        next_exponent = exp_base[(page_head << block_shift) + (safe & bs_mask)];
#pragma unroll
        for (int i = 0; i < G::NV; ++i) {
            const int c = i * kWave + lane;
            const uint32_t r = __shfl(safe, c / G::CPR);
            v[i] = *reinterpret_cast<const u32x4*>(v_base + static_cast<uint64_t>(r) * v_row + (c % G::CPR) * 16);
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
                k16[rt][j] = *reinterpret_cast<const u32x4*>(src + 64 * j + 16 * grp);
            }
            if constexpr (G::N8) k8[rt] = *reinterpret_cast<const u32x2*>(src + 64 * G::N16 + 8 * grp);
        }
    };
    // Tile t; `next_row`: the following tile's rows (`more`: there is one).
    auto compute = [&](bool more, int next_row) __attribute__((always_inline)) {
        const uint32_t valid = next_valid, exponent = next_exponent;
        const bool whole = valid == 0xffffffffu;
#pragma unroll
        for (int i = 0; i < G::NV; ++i) {
            const int c = i * kWave + lane;
            const int row = c / G::CPR;
            const float unit = UnitOf(__shfl(exponent, 32 + row));
            uint4 lo = Widen8<T>(v[i].x, v[i].y, unit);
            uint4 hi = Widen8<T>(v[i].z, v[i].w, unit);
            if (!whole) {  // rows that do not exist: weight 0, but they may hold a NaN
                const uint32_t keep = (valid >> row) & 1u ? ~0u : 0u;
                lo = make_uint4(lo.x & keep, lo.y & keep, lo.z & keep, lo.w & keep);
                hi = make_uint4(hi.x & keep, hi.y & keep, hi.z & keep, hi.w & keep);
            }
            uint4* dst = reinterpret_cast<uint4*>(vs + row * G::RB + (((c % G::CPR) ^ VSwz<D>(row)) * 32));
            dst[0] = lo;
            dst[1] = hi;
        }
        if (more) issue_v(next_row);
        floatx4 s[2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const float unit = UnitOf(__shfl(exponent, 16 * rt + col));
            s[rt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < G::N16; ++j) {
                const u32x4 w = k16[rt][j];
                s[rt] = M::mma(__builtin_bit_cast(vec8, Widen8<T>(w.x, w.y, unit)), qb[2 * j], s[rt]);
                s[rt] = M::mma(__builtin_bit_cast(vec8, Widen8<T>(w.z, w.w, unit)), qb[2 * j + 1], s[rt]);
            }
            if constexpr (G::N8) {
                const u32x2 w = k8[rt];
                s[rt] = M::mma(__builtin_bit_cast(vec8, Widen8<T>(w.x, w.y, unit)), qb[G::NK - 1], s[rt]);
            }
        }
        if (more) issue_k();
        float sv[2][4];
        float mx = neg_inf();
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = s[rt][i] * scale2;
                if (!whole) x = ((valid >> (16 * rt + 4 * grp + i)) & 1u) ? x : neg_inf();
                sv[rt][i] = x;
                mx = fmaxf(mx, x);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(m, mx);
        if (__builtin_amdgcn_ballot_w64(m_new > m) != 0) {
            const float alpha = (m == neg_inf()) ? 0.0f : fast_exp2(m - m_new);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < G::ND; ++dt) o[dt] *= alpha;
            m = m_new;
        }
        const float m_use = (m == neg_inf()) ? 0.0f : m;
        // Weights are summed in fp32 and rounded once to the 16-bit type for PV, off by at most half
        // a step of theirs, as the output is. In fp16 they are scaled by 2^15 (M::kScale, taken back
        // at the end): weights down to 2^-29 then keep all their bits, and those that vanish are
        // below 2^-39.
        float pr[2][4];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = fast_exp2(sv[rt][i] - m_use);
                l += w;
                pr[rt][i] = w * M::kScale;
            }
        }
        const vec8 pb = __builtin_bit_cast(
            vec8, make_uint4(M::pack(pr[0][0], pr[0][1]), M::pack(pr[0][2], pr[0][3]),
                             M::pack(pr[1][0], pr[1][1]), M::pack(pr[1][2], pr[1][3])));
        // The tile is this wave's own: its LDS writes and reads stay in order without a barrier.
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
        for (int dt = 0; dt < G::ND; ++dt) {
            const uint8_t* a = vs + tr_rd + ((dt * 32) ^ tr_x);
            const uint2 lo = M::Tr::read(a);
            const uint2 hi = M::Tr::read(a + 16 * G::RB);
            o[dt] = M::mma(__builtin_bit_cast(vec8, make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, o[dt]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    int tile = kWaveHeads ? 0 : wave;
    if (tile < n_tiles) {
        issue_v(row_of(tile));
        issue_k();
    }
    int row = row_of(tile + TS);
    for (; tile < n_tiles; tile += TS) {
        const int now = row;
        row = row_of(tile + 2 * TS);
        compute(tile + TS < n_tiles, now);
    }

    if constexpr (M::kScale != 1.0f) {
#pragma unroll
        for (int dt = 0; dt < G::ND; ++dt) o[dt] *= 1.0f / M::kScale;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const bool direct = p.num_splits == 1;
    if constexpr (kWaveHeads) {
        if (!slot_ok || col >= hc) return;
        const int64_t hq = h0 + col;
        if (direct) {
            const float inv = l > 0.0f ? 1.0f / l : l;
            uint16_t* out = static_cast<uint16_t*>(p.out) + b * p.o_sb + hq * p.o_sh;
#pragma unroll
            for (int dt = 0; dt < G::ND; ++dt) {
                *reinterpret_cast<uint2*>(out + dt * 16 + 4 * grp) =
                    make_uint2(M::pack(o[dt][0] * inv, o[dt][1] * inv), M::pack(o[dt][2] * inv, o[dt][3] * inv));
            }
        } else {
            const int64_t flat = (b * p.num_heads + hq) * p.num_splits + split;
#pragma unroll
            for (int dt = 0; dt < G::ND; ++dt) {
                *reinterpret_cast<floatx4*>(p.partial_o + flat * D + dt * 16 + 4 * grp) = o[dt];
            }
            if (grp == 0) {
                p.partial_m[flat] = (m == neg_inf()) ? neg_inf() : m * kLn2;
                p.partial_l[flat] = l;
            }
        }
        return;
    }
    // Wave states to LDS, then one thread per (head, dim) merges the four waves.
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(s_v);  // [wave][head][D]
#pragma unroll
    for (int dt = 0; dt < G::ND; ++dt) {
        *reinterpret_cast<floatx4*>(s_o + (wave * kMfmaHeads + col) * D + dt * 16 + 4 * grp) = o[dt];
    }
    if (grp == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < hc * D; idx += kDecodeThreads) {
        const int h = idx / D;
        const int d = idx % D;
        float mm = neg_inf();
#pragma unroll
        for (int w = 0; w < kDecodeWaves; ++w) mm = fmaxf(mm, s_m[w][h]);
        float lsum = 0.0f, osum = 0.0f;
        // (also where no wave has a maximum: a NaN among the scores must not become a zero)
#pragma unroll
        for (int w = 0; w < kDecodeWaves; ++w) {
            const float mw = s_m[w][h];
            const float wgt = mw == neg_inf() ? 0.0f : fast_exp2(mw - mm);
            lsum += s_l[w][h] * wgt;
            osum += s_o[(w * kMfmaHeads + h) * D + d] * wgt;
        }
        const int64_t hq = h0 + h;
        if (direct) {
            const float inv = lsum > 0.0f ? 1.0f / lsum : lsum;
            uint8_t* out_row = static_cast<uint8_t*>(p.out) + (b * p.o_sb + hq * p.o_sh) * 2;
            E::Dec::store1(out_row, d, osum * inv);
        } else {
            const int64_t flat = (b * p.num_heads + hq) * p.num_splits + split;
            p.partial_o[flat * D + d] = osum;
            if (d == 0) {
                p.partial_m[flat] = (mm == neg_inf()) ? neg_inf() : mm * kLn2;
                p.partial_l[flat] = lsum;
            }
        }
    }
}

struct Dec8F16 {
    using Type = F16;
    using Dec = DecF16;
};
struct Dec8BF16 {
    using Type = BF16;
    using Dec = DecBF16;
};

template <typename E, int D>
int LaunchDecode8(const sca_decode8_params& p8, hipStream_t s) {
    sca_decode_params q = p8.base;
    int block_shift = 0;
    while ((int64_t{1} << block_shift) < q.block_size) ++block_shift;
    if (q.seq_lens == nullptr || q.batch <= kRankBatch || q.batch > kMaxOrderedBatch) q.batch_order = nullptr;
    if (q.batch_order != nullptr) {
        hipLaunchKernelGGL(decode_order_kernel, dim3(static_cast<unsigned>((q.batch + 255) / 256)), dim3(256),
                           0, s, q.seq_lens, static_cast<int>(q.batch), q.batch_order);
        if (const int rc = CheckLaunch("decode_order_kernel", s)) return rc;
    }
    const int64_t group = q.num_heads / q.num_kv_heads;
    const int h_chunks = static_cast<int>((group + kMfmaHeads - 1) / kMfmaHeads);
    const int64_t slots = q.num_kv_heads * h_chunks;
    if (q.slot_waves != kDecodeWaves) {
        const dim3 grid(static_cast<unsigned>(q.num_splits),
                        static_cast<unsigned>((slots + kDecodeWaves - 1) / kDecodeWaves),
                        static_cast<unsigned>(q.batch));
        hipLaunchKernelGGL((decode8_kernel<E, D, true>), grid, dim3(kDecodeThreads), 0, s, q, p8.k_exp,
                           p8.v_exp, h_chunks, block_shift);
    } else {
        const dim3 grid(static_cast<unsigned>(q.num_splits), static_cast<unsigned>(slots),
                        static_cast<unsigned>(q.batch));
        hipLaunchKernelGGL((decode8_kernel<E, D, false>), grid, dim3(kDecodeThreads), 0, s, q, p8.k_exp,
                           p8.v_exp, h_chunks, block_shift);
    }
    int rc = CheckLaunch("decode8_kernel", s);
    if (rc != 0 || q.num_splits == 1) return rc;
    const int64_t threads = q.batch * q.num_heads * (D / 4);
    const unsigned blocks = static_cast<unsigned>((threads + kCombineThreads - 1) / kCombineThreads);
    hipLaunchKernelGGL((decode_combine_kernel<typename E::Dec, D>), dim3(blocks), dim3(kCombineThreads), 0, s,
                       q);
    return CheckLaunch("decode_combine_kernel", s);
}

template <typename E>
int LaunchDecode8For(const sca_decode8_params& p, hipStream_t s) {
    switch (p.base.head_dim) {
        case 32: return LaunchDecode8<E, 32>(p, s);
        case 64: return LaunchDecode8<E, 64>(p, s);
        case 96: return LaunchDecode8<E, 96>(p, s);
        case 128: return LaunchDecode8<E, 128>(p, s);
        case 160: return LaunchDecode8<E, 160>(p, s);
        case 192: return LaunchDecode8<E, 192>(p, s);
        case 256: return LaunchDecode8<E, 256>(p, s);
        default: break;
    }
    return SetError(SCA_E_UNSUPPORTED_HEAD_DIM,
                    "decode8: head_dim=" + std::to_string(p.base.head_dim) + " is not instantiated");
}

int ValidateDecode8(const sca_decode8_params* p8) {
    if (p8 == nullptr) return SetError(SCA_E_SHAPE_MISMATCH, "decode8: null params");
    const sca_decode_params* p = &p8->base;
    if (p->q == nullptr || p->k == nullptr || p->v == nullptr || p->out == nullptr ||
        p8->k_exp == nullptr || p8->v_exp == nullptr || p->page_table == nullptr) {
        return SetError(SCA_E_SHAPE_MISMATCH, "decode8: null pointer");
    }
    if (p->num_splits < 1 || p->num_splits > 65535) {
        return SetError(SCA_E_SHAPE_MISMATCH,
                        "decode8: num_splits=" + std::to_string(p->num_splits) + " is not in [1, 65535]");
    }
    if (p->num_splits > 1 &&
        (p->partial_m == nullptr || p->partial_l == nullptr || p->partial_o == nullptr)) {
        return SetError(SCA_E_WORKSPACE, "decode8: num_splits > 1 needs partial_m/l/o scratch");
    }
    if (p->batch < 1 || p->batch > 65535 || p->num_heads < 1 || p->num_heads > 65535 ||
        p->num_kv_heads < 1 || p->num_heads % p->num_kv_heads != 0) {
        return SetError(SCA_E_SHAPE_MISMATCH,
                        "decode8: invalid heads (H_q=" + std::to_string(p->num_heads) +
                            ", H_kv=" + std::to_string(p->num_kv_heads) + ") or batch");
    }
    if (p->seq_kv < 0) return SetError(SCA_E_SHAPE_MISMATCH, "decode8: seq_kv < 0");
    if (p->seq_kv > 0x7fffffff - 4096) {
        return SetError(SCA_E_SEQ_TOO_LONG, "decode8: seq_kv=" + std::to_string(p->seq_kv));
    }
    if (p->dtype != SCA_DTYPE_F16 && p->dtype != SCA_DTYPE_BF16) {
        return SetError(SCA_E_UNSUPPORTED_DTYPE,
                        "decode8: queries are fp16 or bf16; dtype id " + std::to_string(p->dtype));
    }
    if (p->block_size < 8 || (p->block_size & (p->block_size - 1)) != 0 || p->max_blocks_per_seq <= 0 ||
        p->num_kv_blocks <= 0 || p->num_kv_blocks > 0x7fffffffLL / p->block_size) {
        return SetError(SCA_E_SHAPE_MISMATCH,
                        "decode8: block_size must be a power of two of at least 8, max_blocks_per_seq and "
                        "num_kv_blocks positive, and the pool's tokens below 2^31");
    }
    if (!Aligned16(p->q) || !Aligned16(p->k) || !Aligned16(p->v) || !Aligned16(p->out) || p->q_sb % 8 ||
        p->q_sh % 8 || p->o_sb % 8 || p->o_sh % 8 || p->k_sh % 16 || p->k_ss % 16 || p->v_sh % 16 ||
        p->v_ss % 16 || p->k_ss < 0 || p->k_ss > 0x7fffffff || p->v_ss < 0 || p->v_ss > 0x7fffffff) {
        return SetError(SCA_E_LAYOUT_MISMATCH,
                        "decode8: pointers must be 16 B aligned, strides multiples of 16 B, row strides from 0 to 2^31");
    }
    if (p->slot_waves != 0 && p->slot_waves != 1 && p->slot_waves != kDecodeWaves) {
        return SetError(SCA_E_SHAPE_MISMATCH,
                        "decode8: slot_waves must be 0, 1 or 4; got " + std::to_string(p->slot_waves));
    }
    if ((reinterpret_cast<uintptr_t>(p->batch_order) & 7u) != 0) {
        return SetError(SCA_E_LAYOUT_MISMATCH, "decode8: batch_order must be 8 B aligned");
    }
    return 0;
}

}  // namespace
}  // namespace sca_hip

extern "C" {

int sca_hip_decode8_paged(const sca_decode8_params* params, void* stream) {
    if (const int rc = sca_hip::ValidateDecode8(params)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return params->base.dtype == SCA_DTYPE_F16 ? sca_hip::LaunchDecode8For<sca_hip::Dec8F16>(*params, s)
                                               : sca_hip::LaunchDecode8For<sca_hip::Dec8BF16>(*params, s);
}

}  // extern "C"
