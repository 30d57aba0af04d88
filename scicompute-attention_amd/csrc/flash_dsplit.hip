// ============================================================================================
// Split-dims kernel (head_dim 192 and 256): one wave per SIMD, 64 query rows per wave pair.
//
// Why: 64 rows x 256 dims of O and Q are 384 registers a lane, so the wide kernel's wave (64 rows,
// all dims) does not fit, and a wave of 32 rows reads every fragment from LDS for one MFMA, which
// bounds it. Here the two waves of a 64-row group share the rows differently in the two products:
//   QK, softmax: wave dh owns subtile dh (32 rows) and computes its scores for all 32 keys of a
//                tile, so the row state (m, l) stays in one wave;
//   PV:          wave dh owns dims [dh*D/2, +D/2) of all 64 rows, so every transposed V fragment
//                (the slow LDS reads) feeds two MFMAs. Its own subtile's P comes from registers,
//                the partner's through LDS (2 KB per wave and tile).
// O (64 rows x D/2) and Q (32 rows x D) take 192 AGPRs at D = 256.
//
// Pipeline, step t: QK of tile t+2, softmax of tile t+1, PV of tile t, one barrier. A move of the
// running max for tile u is decided by the owner at the end of step u-2, published as 32 factors
// and a flag that holds u, and applied by both waves to O at the end of step u-1 (after PV(u-1)).
// K and V tiles (32 keys) come by buffer->LDS DMA into rings of four slots each; loads past the
// last tile are out of the resource's range and cost no traffic, so every step issues the same
// number and waits on the same count. As in the wide kernel the order inside a step is explicit and
// hazards the compiler cannot see (inline-asm MFMAs and LDS reads) are covered where they arise.
//
// Measured (MI355X) against the register-staged kernel that served these head dims before: D = 256,
// 16 heads x 4096 keys causal 325 -> 139 us (423 -> 992 TF/s), 2 x 16 heads non-causal 1,279 ->
// 504 us (1,090); D = 192, 2 x 16 heads causal 454 -> 220 us (939), non-causal 849 -> 422 (976);
// short sequences too (8 heads x 300 keys, D = 256: 27 -> 16 us).
// ============================================================================================

#include <hip/hip_runtime.h>

#include <string>
#include <type_traits>

#include "flash_common.hpp"

namespace sca_hip {
namespace {

// kCut: rows packed and / or keys split (SplitArgs).
template <typename E, int D, bool kCausal, bool kCut, Denominator kDen>
__global__ __launch_bounds__(DsplitGeom<D>::THREADS, 1) void flash_fwd_dsplit_kernel(
    const sca_flash_params p, int num_q_tiles, const SplitArgs sp) {
    constexpr bool kPaged = false;
    const PagedJob job{};
#include "flash_dsplit_body.hpp"
}

}  // namespace

template <typename E, int D, bool kCausal>
int LaunchFlashDsplit(const sca_flash_params& p, const SplitArgs& sp, hipStream_t s) {
    using G = DsplitGeom<D>;
    const int64_t num_q_tiles = (p.seq_q * sp.pack + G::BM - 1) / G::BM;
    const int64_t blocks = num_q_tiles * p.batch * (p.num_heads / sp.pack) * sp.splits;
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffffLL) {
        return SetError(SCA_E_SEQ_TOO_LONG, "flash: grid of " + std::to_string(blocks) +
                                                " workgroups exceeds the launch limit");
    }
    auto launch = [&]<bool kCut, Denominator kDen>() -> int {
        if (const int rc = EnsureLdsLimit<&flash_fwd_dsplit_kernel<E, D, kCausal, kCut, kDen>>(
                G::LDS_BYTES, "flash LDS limit")) {
            return rc;
        }
        hipLaunchKernelGGL((flash_fwd_dsplit_kernel<E, D, kCausal, kCut, kDen>),
                           dim3(static_cast<unsigned>(blocks)), dim3(G::THREADS), G::LDS_BYTES, s, p,
                           static_cast<int>(num_q_tiles), sp);
        return CheckLaunch("flash_fwd_dsplit_kernel", s);
    };
    const bool cut = sp.pack != 1 || sp.splits != 1;
    if (p.lse != nullptr) {
        constexpr Denominator kDen = DenominatorFor<D>(true);
        return cut ? launch.template operator()<true, kDen>() : launch.template operator()<false, kDen>();
    }
    constexpr Denominator kDen = DenominatorFor<D>(false);
    return cut ? launch.template operator()<true, kDen>() : launch.template operator()<false, kDen>();
}

#define SCA_INSTANTIATE(E, D)                                                     \
    template int LaunchFlashDsplit<E, D, false>(const sca_flash_params&, const SplitArgs&, hipStream_t); \
    template int LaunchFlashDsplit<E, D, true>(const sca_flash_params&, const SplitArgs&, hipStream_t);
SCA_INSTANTIATE(F16, 192)
SCA_INSTANTIATE(F16, 256)
SCA_INSTANTIATE(BF16, 192)
SCA_INSTANTIATE(BF16, 256)

}  // namespace sca_hip
