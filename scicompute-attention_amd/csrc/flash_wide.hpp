// ============================================================================================
// Wide-row kernel (head_dim 32, 64, 96, 128 and 160): one wave per SIMD and 64 query rows per wave.
//
// Why: the fragment reads from LDS are what bounds the 32-row kernels. Every K fragment (32 keys x
// 16 dims) and every V^T fragment feeds one MFMA per 32 query rows a wave holds, and the
// transposed V reads stream at about half the rate of ds_read_b128. With 64 rows per wave each
// fragment feeds two MFMAs, which halves the LDS bytes per FLOP. 64 rows need about 220 VGPRs
// plus 64 (D = 64) to 160 (D = 160) accumulator registers for O and half as many for Q, which only
// one wave per SIMD has (two up to D = 64); that wave then has to overlap its own VALU work with
// its MFMAs. It does when O lives in AGPRs and the instruction stream alternates one MFMA with a
// few VALU instructions, so the step below is written in an explicit order: every MFMA, fragment
// read and wait is an inline asm statement, the C++ VALU code between them is fenced with
// sched_barrier, and the data hazards the compiler cannot see are covered by waits stated at each
// use (see the step). D = 160 fills the register file (240 AGPRs) and the LDS (160 KB).
//
// Workgroup: 4 waves = 2 row groups (64 rows each, two 32-row subtiles) x 2 key halves (32 keys
// of every 64-key tile); K and V tiles come by buffer->LDS DMA into rings of four slots each,
// three tiles ahead. The two key halves of a row group are merged through LDS at the end.
//
// Measured (MI355X, 2 x 16 heads x 4096 keys) against the register-staged kernel that served these
// head dims before: D = 160 causal 398 -> 173 us (432 -> 996 TF/s), non-causal 723 -> 333 us (1,032);
// D = 96 causal 175 -> 122 us (847), non-causal 315 -> 221 us (932); D = 32 causal 78 -> 57 us,
// non-causal 141 -> 102 us (672: the softmax VALU bounds it, at 4 MFMAs per 48 VALU operations).
//
// With one workgroup per CU (from D = 96 on) its fixed part is not hidden: 8,192 workgroups of one key tile (D = 128)
// took 322 us, 9.2 us each beside the step; with the K/V DMAs ahead of the wait for Q, 32-bit index
// arithmetic, no rescale of the zero O and both key halves sharing the merge and the stores 246 us.
// ============================================================================================

#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "flash_common.hpp"

namespace sca_hip {
namespace {

// kMode: plain, packed varlen, cut (rows packed and / or keys split: SplitArgs), or paged (PagedJob:
// packed rows of one sequence over the pages of its keys).
enum WideMode { kPlain, kPackedVarlen, kCut, kPaged };

template <typename E, int D, bool kCausal, WideMode kMode, Denominator kDen>
__global__ __launch_bounds__(WideGeom<D>::THREADS, 1) void flash_fwd_wide_kernel(
    const sca_flash_params p, int num_q_tiles, const VarlenArgs vl, const SplitArgs sp) {
    const PagedJob job{};
#include "flash_wide_body.hpp"
}

}  // namespace

template <typename E, int D, bool kCausal>
int LaunchFlashWide(const sca_flash_params& p, const SplitArgs& sp, hipStream_t s) {
    using G = WideGeom<D>;
    const int64_t num_q_tiles = (p.seq_q * sp.pack + G::BM - 1) / G::BM;
    const int64_t blocks = num_q_tiles * p.batch * (p.num_heads / sp.pack) * sp.splits;
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL) {
        return SetError(SCA_E_SEQ_TOO_LONG, "flash: grid of " + std::to_string(blocks) +
                                                " workgroups exceeds the launch limit");
    }
    auto launch = [&]<WideMode kMode, Denominator kDen>() -> int {
        if (const int rc = EnsureLdsLimit<&flash_fwd_wide_kernel<E, D, kCausal, kMode, kDen>>(
                G::LDS_BYTES, "flash LDS limit")) {
            return rc;
        }
        hipLaunchKernelGGL((flash_fwd_wide_kernel<E, D, kCausal, kMode, kDen>),
                           dim3(static_cast<unsigned>(blocks)), dim3(G::THREADS), G::LDS_BYTES, s, p,
                           static_cast<int>(num_q_tiles), VarlenArgs{nullptr, nullptr, nullptr}, sp);
        return CheckLaunch("flash_fwd_wide_kernel", s);
    };
    const bool cut = sp.pack != 1 || sp.splits != 1;
    if (p.lse != nullptr) {
        constexpr Denominator kDen = DenominatorFor<D>(true);
        return cut ? launch.template operator()<kCut, kDen>() : launch.template operator()<kPlain, kDen>();
    }
    constexpr Denominator kDen = DenominatorFor<D>(false);
    return cut ? launch.template operator()<kCut, kDen>() : launch.template operator()<kPlain, kDen>();
}

// One launch over a packed batch: the wide kernel, one workgroup per (work entry, head).
template <typename E, int D, bool kCausal>
int LaunchFlashVarlen(const sca_flash_varlen_params& v, hipStream_t s) {
    using G = WideGeom<D>;
    static_assert(G::BM == 128, "the work list's row tiles are 128 rows");
    static_assert(DenominatorFor<D>(false) == kUnrounded);
    // 32-bit buffer offsets: a sequence's rows plus the wide kernel's ring overrun must fit.
    const int64_t rows_k = v.max_seq_kv + 8 * G::BN;
    if (rows_k * v.k_ss * 2 >= (1LL << 31) || rows_k * v.v_ss * 2 >= (1LL << 31)) {
        return SetError(SCA_E_SEQ_TOO_LONG, "flash varlen: a sequence of " +
                                                std::to_string(v.max_seq_kv) +
                                                " keys exceeds the 32-bit tile offsets");
    }
    const int64_t blocks = v.num_tiles * v.num_heads;
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL) {
        return SetError(SCA_E_SEQ_TOO_LONG, "flash varlen: grid too large");
    }
    sca_flash_params p{};
    p.q = v.q;
    p.k = v.k;
    p.v = v.v;
    p.out = v.out;
    p.lse = nullptr;
    p.batch = 1;
    p.num_heads = v.num_heads;
    p.num_kv_heads = v.num_kv_heads;
    p.head_dim = v.head_dim;
    p.q_sh = v.q_sh, p.q_ss = v.q_ss;
    p.k_sh = v.k_sh, p.k_ss = v.k_ss;
    p.v_sh = v.v_sh, p.v_ss = v.v_ss;
    p.o_sh = v.o_sh, p.o_ss = v.o_ss;
    p.scale = v.scale;
    p.causal = v.causal;
    p.dtype = v.dtype;
    if (const int rc = EnsureLdsLimit<&flash_fwd_wide_kernel<E, D, kCausal, kPackedVarlen, kUnrounded>>(
            G::LDS_BYTES, "flash LDS limit")) {
        return rc;
    }
    hipLaunchKernelGGL((flash_fwd_wide_kernel<E, D, kCausal, kPackedVarlen, kUnrounded>),
                       dim3(static_cast<unsigned>(blocks)), dim3(G::THREADS), G::LDS_BYTES, s, p,
                       0, VarlenArgs{v.cu_seqlens_q, v.cu_seqlens_kv, v.tiles},
                       SplitArgs{1, 1, nullptr, nullptr});
    return CheckLaunch("flash_fwd_wide_kernel (varlen)", s);
}

}  // namespace sca_hip
