// Data movement of a paged KV cache that keeps K and V in 8 bits (e4m3.hpp): codes
// [num_blocks][block_size][H_kv][D], one byte a value, and exponent bytes
// [num_blocks][H_kv][block_size], so that the attention kernels fetch the exponents of a page's
// tokens for their head as neighbouring bytes.
//
// All three kernels move bytes and compute next to nothing; HBM bounds them. Eight values a lane (16 bytes
// read, 8 written) and a token and head on 4 to 32 lanes, so that a row's maximum is a few shuffles.
// Measured (MI355X), bf16, 8 KV heads: 8,400 tokens of D 128 stored in 13.3 us (51 MB, 3.9 TB/s) and read back
// in twice 7.0 (26 MB each, 3.7 TB/s); 30,001 of D 96 30.2 (137 MB, 4.6) and twice 13.1 (70 MB, 5.3).

#include <hip/hip_runtime.h>

#include <string>

#include "e4m3.hpp"
#include "sca_device.hpp"

namespace sca_hip {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 65535;

// Largest |x| over the LPR lanes of a row (LPR a power of two up to 32).
template <int LPR>
__device__ __forceinline__ float RowMax(float x) {
#pragma unroll
    for (int off = 1; off < LPR; off *= 2) x = fmaxf(x, __shfl_xor(x, off));
    return x;
}

// One row of D values (a token's K or V of one head) on LPR lanes, eight values a lane: quantises it
// and writes codes and exponent. Lanes past D/8 hold zeros and write nothing.
template <typename E, int D, int LPR>
__device__ __forceinline__ void HoldRow(const uint4& raw, int sub, uint8_t* codes, uint8_t* exponent) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = E::to_float(static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2))));
        // (comparisons, not fmin / fmax: a NaN passes through them, and fmaxf below leaves it out)
        x[i] = v > Held<E>::kLargest ? Held<E>::kLargest : v < -Held<E>::kLargest ? -Held<E>::kLargest : v;
        a = fmaxf(a, fabsf(x[i]));
    }
    const uint32_t e = ExponentFor(RowMax<LPR>(a));
    const float inv = InverseUnit(e);
    if (sub * 8 < D) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        *reinterpret_cast<uint2*>(codes + sub * 8) =
            make_uint2(Codes4(x[0], x[1], x[2], x[3]), Codes4(x[4], x[5], x[6], x[7]));
    }
    if (sub == 0) *exponent = static_cast<uint8_t>(e);
}

// A row group of LPR lanes per (token, head): both its rows (K, V) are fetched before either is
// reduced, so that a lane has two loads in flight.
template <typename E, int D>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(
    uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes, uint8_t* __restrict__ k_exp,
    uint8_t* __restrict__ v_exp, const uint16_t* __restrict__ k_new, const uint16_t* __restrict__ v_new,
    const int32_t* __restrict__ slots, int64_t num_rows, uint32_t heads, uint32_t block_size,
    int64_t num_blocks) {
    constexpr int LPR = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
    constexpr int kRows = kThreads / LPR;
    const int sub = threadIdx.x % LPR;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / LPR; r < num_rows;
         r += stride) {
        const int64_t t = num_rows <= 0xffffffffLL ? static_cast<uint32_t>(r) / heads : r / heads;
        const uint32_t h = static_cast<uint32_t>(r - t * heads);
        const int32_t slot = slots[t];
        if (slot < 0 || static_cast<uint32_t>(slot) / block_size >= num_blocks) continue;
        uint4 kr = make_uint4(0, 0, 0, 0), vr = kr;
        if (sub * 8 < D) {
            kr = *reinterpret_cast<const uint4*>(k_new + r * D + sub * 8);
            vr = *reinterpret_cast<const uint4*>(v_new + r * D + sub * 8);
        }
        const uint32_t page = static_cast<uint32_t>(slot) / block_size;
        const uint32_t off = static_cast<uint32_t>(slot) - page * block_size;
        const int64_t row = (static_cast<int64_t>(slot) * heads + h) * D;
        const int64_t at = (static_cast<int64_t>(page) * heads + h) * block_size + off;
        HoldRow<E, D, LPR>(kr, sub, k_codes + row, k_exp + at);
        HoldRow<E, D, LPR>(vr, sub, v_codes + row, v_exp + at);
    }
}

// Pages read back: 16 codes a lane. Ids outside the pool give zeros.
template <typename E>
__global__ __launch_bounds__(kThreads) void kv8_gather_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents,
    const int32_t* __restrict__ ids, int64_t n_ids, uint4* __restrict__ out, uint32_t heads,
    uint32_t row_chunks, uint32_t block_size, int64_t num_blocks) {
    const uint32_t page_chunks = block_size * heads * row_chunks;
    const int64_t total = n_ids * page_chunks;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += stride) {
        const int64_t n = total <= 0xffffffffLL ? static_cast<uint32_t>(i) / page_chunks : i / page_chunks;
        const uint32_t c = static_cast<uint32_t>(i - n * page_chunks);
        const int64_t page = ids[n];
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (page >= 0 && page < num_blocks) {
            const uint32_t row = c / row_chunks;
            const uint32_t t = row / heads;
            const uint32_t h = row - t * heads;
            const uint4 w = *reinterpret_cast<const uint4*>(codes + (page * page_chunks + c) * 16);
            const float unit = UnitOf(exponents[(page * heads + h) * block_size + t]);
            lo = Widen8<E>(w.x, w.y, unit);
            hi = Widen8<E>(w.z, w.w, unit);
        }
        out[2 * i] = lo;
        out[2 * i + 1] = hi;
    }
}

__global__ __launch_bounds__(kThreads) void kv8_reset_kernel(
    uint4* __restrict__ k_codes, uint4* __restrict__ v_codes, uint2* __restrict__ k_exp,
    uint2* __restrict__ v_exp, const int32_t* __restrict__ ids, int64_t n_ids, uint32_t page_chunks,
    uint32_t exp_chunks, int64_t num_blocks) {
    const int64_t total = n_ids * page_chunks;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += stride) {
        const int64_t n = i / page_chunks;
        const uint32_t c = static_cast<uint32_t>(i - n * page_chunks);
        const int64_t page = ids[n];
        if (page < 0 || page >= num_blocks) continue;
        k_codes[page * page_chunks + c] = make_uint4(0, 0, 0, 0);
        v_codes[page * page_chunks + c] = make_uint4(0, 0, 0, 0);
        if (c < exp_chunks) {  // (8 exponents for every 16 * D codes or fewer: always fewer chunks)
            k_exp[page * exp_chunks + c] = make_uint2(0, 0);
            v_exp[page * exp_chunks + c] = make_uint2(0, 0);
        }
    }
}

unsigned GridFor(int64_t total, int64_t per_block) {
    int64_t blocks = (total + per_block - 1) / per_block;
    if (blocks < 1) blocks = 1;
    if (blocks > kMaxGrid) blocks = kMaxGrid;
    return static_cast<unsigned>(blocks);
}

bool AlignedTo(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int CheckShape8(const sca_kv_shape* shape, const char* what) {
    if (shape == nullptr) return SetError(SCA_E_SHAPE_MISMATCH, std::string(what) + ": null shape");
    if (shape->num_blocks <= 0 || shape->block_size <= 0 || shape->num_kv_heads <= 0 ||
        shape->head_dim <= 0) {
        return SetError(SCA_E_SHAPE_MISMATCH, std::string(what) + ": non-positive KV geometry");
    }
    const int64_t d = shape->head_dim;
    if (d % 32 != 0 || d > 256 || d == 224) {
        return SetError(SCA_E_UNSUPPORTED_HEAD_DIM, std::string(what) + ": head_dim=" + std::to_string(d) +
                                                        " (8-bit pages: 32, 64, 96, 128, 160, 192, 256)");
    }
    if (shape->block_size % 8 != 0) {
        return SetError(SCA_E_SHAPE_MISMATCH, std::string(what) + ": block_size=" +
                                                  std::to_string(shape->block_size) +
                                                  " (8-bit pages hold multiples of 8 tokens)");
    }
    // Positions inside a page, and slots, are 32-bit numbers in the kernels.
    if (shape->num_kv_heads > 65535 ||
        shape->block_size > 0x7fffffffLL / (shape->num_kv_heads * d) ||
        shape->num_blocks > 0x7fffffffLL / shape->block_size) {
        return SetError(SCA_E_SHAPE_MISMATCH, std::string(what) + ": a page or the pool passes 2^31");
    }
    return 0;
}

int CheckLayer8(const sca_kv8_layer* layer, const char* what) {
    if (layer == nullptr || layer->k == nullptr || layer->v == nullptr || layer->k_exp == nullptr ||
        layer->v_exp == nullptr) {
        return SetError(SCA_E_SHAPE_MISMATCH, std::string(what) + ": null pointer");
    }
    if (!AlignedTo(layer->k, 16) || !AlignedTo(layer->v, 16) || !AlignedTo(layer->k_exp, 8) ||
        !AlignedTo(layer->v_exp, 8)) {
        return SetError(SCA_E_LAYOUT_MISMATCH,
                        std::string(what) + ": codes must be 16 B and exponents 8 B aligned");
    }
    return 0;
}

template <typename E, int D>
int LaunchAppend(const sca_kv8_layer& l, const void* k_new, const void* v_new, const int32_t* slots,
                 int64_t num_tokens, const sca_kv_shape& shape, hipStream_t s) {
    constexpr int LPR = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
    const int64_t rows = num_tokens * shape.num_kv_heads;
    hipLaunchKernelGGL((kv8_append_kernel<E, D>), dim3(GridFor(rows, kThreads / LPR)), dim3(kThreads), 0, s,
                       static_cast<uint8_t*>(l.k), static_cast<uint8_t*>(l.v), l.k_exp, l.v_exp,
                       static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), slots,
                       rows, static_cast<uint32_t>(shape.num_kv_heads),
                       static_cast<uint32_t>(shape.block_size), shape.num_blocks);
    return CheckLaunch("kv8_append_kernel", s);
}

template <typename E>
int AppendFor(const sca_kv8_layer& l, const void* k_new, const void* v_new, const int32_t* slots,
              int64_t num_tokens, const sca_kv_shape& shape, hipStream_t s) {
    switch (shape.head_dim) {
        case 32: return LaunchAppend<E, 32>(l, k_new, v_new, slots, num_tokens, shape, s);
        case 64: return LaunchAppend<E, 64>(l, k_new, v_new, slots, num_tokens, shape, s);
        case 96: return LaunchAppend<E, 96>(l, k_new, v_new, slots, num_tokens, shape, s);
        case 128: return LaunchAppend<E, 128>(l, k_new, v_new, slots, num_tokens, shape, s);
        case 160: return LaunchAppend<E, 160>(l, k_new, v_new, slots, num_tokens, shape, s);
        case 192: return LaunchAppend<E, 192>(l, k_new, v_new, slots, num_tokens, shape, s);
        default: return LaunchAppend<E, 256>(l, k_new, v_new, slots, num_tokens, shape, s);
    }
}

int CheckType16(int32_t dtype, const char* what) {
    if (dtype == SCA_DTYPE_F16 || dtype == SCA_DTYPE_BF16) return 0;
    return SetError(SCA_E_UNSUPPORTED_DTYPE, std::string(what) + ": 8-bit pages stand for fp16 or bf16; dtype id " +
                                                 std::to_string(dtype));
}

}  // namespace
}  // namespace sca_hip

using sca_hip::SetError;

extern "C" {

int sca_hip_kv8_append(const sca_kv8_layer* layer, const void* k_new, const void* v_new,
                       const int32_t* slot_mapping, int64_t num_tokens, const sca_kv_shape* shape,
                       int32_t dtype, void* stream) {
    int rc = sca_hip::CheckShape8(shape, "kv8_append");
    if (rc == 0) rc = sca_hip::CheckType16(dtype, "kv8_append");
    if (rc != 0) return rc;
    if (num_tokens <= 0) return 0;
    rc = sca_hip::CheckLayer8(layer, "kv8_append");
    if (rc != 0) return rc;
    if (k_new == nullptr || v_new == nullptr || slot_mapping == nullptr) {
        return SetError(SCA_E_SHAPE_MISMATCH, "kv8_append: null pointer");
    }
    if (!sca_hip::AlignedTo(k_new, 16) || !sca_hip::AlignedTo(v_new, 16)) {
        return SetError(SCA_E_LAYOUT_MISMATCH, "kv8_append: k_new and v_new must be 16 B aligned");
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SCA_DTYPE_F16
               ? sca_hip::AppendFor<sca_hip::F16>(*layer, k_new, v_new, slot_mapping, num_tokens, *shape, s)
               : sca_hip::AppendFor<sca_hip::BF16>(*layer, k_new, v_new, slot_mapping, num_tokens, *shape, s);
}

int sca_hip_kv8_reset_blocks(const sca_kv8_layer* layer, const int32_t* block_ids, int64_t num_block_ids,
                             const sca_kv_shape* shape, void* stream) {
    int rc = sca_hip::CheckShape8(shape, "kv8_reset");
    if (rc != 0) return rc;
    if (num_block_ids <= 0) return 0;
    rc = sca_hip::CheckLayer8(layer, "kv8_reset");
    if (rc != 0) return rc;
    if (block_ids == nullptr) return SetError(SCA_E_SHAPE_MISMATCH, "kv8_reset: null pointer");
    const int64_t page_chunks = shape->block_size * shape->num_kv_heads * shape->head_dim / 16;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(sca_hip::kv8_reset_kernel,
                       dim3(sca_hip::GridFor(num_block_ids * page_chunks, sca_hip::kThreads)),
                       dim3(sca_hip::kThreads), 0, s, static_cast<uint4*>(layer->k),
                       static_cast<uint4*>(layer->v), reinterpret_cast<uint2*>(layer->k_exp),
                       reinterpret_cast<uint2*>(layer->v_exp), block_ids, num_block_ids,
                       static_cast<uint32_t>(page_chunks),
                       static_cast<uint32_t>(shape->block_size * shape->num_kv_heads / 8),
                       shape->num_blocks);
    return sca_hip::CheckLaunch("kv8_reset_kernel", s);
}

int sca_hip_kv8_gather(const void* codes, const uint8_t* exponents, const int32_t* block_ids,
                       int64_t num_block_ids, void* out, const sca_kv_shape* shape, int32_t dtype,
                       void* stream) {
    int rc = sca_hip::CheckShape8(shape, "kv8_gather");
    if (rc == 0) rc = sca_hip::CheckType16(dtype, "kv8_gather");
    if (rc != 0) return rc;
    if (num_block_ids <= 0) return 0;
    if (codes == nullptr || exponents == nullptr || block_ids == nullptr || out == nullptr) {
        return SetError(SCA_E_SHAPE_MISMATCH, "kv8_gather: null pointer");
    }
    if (!sca_hip::AlignedTo(codes, 16) || !sca_hip::AlignedTo(out, 16)) {
        return SetError(SCA_E_LAYOUT_MISMATCH, "kv8_gather: buffers must be 16 B aligned");
    }
    const int64_t chunks = num_block_ids * shape->block_size * shape->num_kv_heads * shape->head_dim / 16;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(sca_hip::GridFor(chunks, sca_hip::kThreads));
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(sca_hip::kThreads), 0, s, static_cast<const uint8_t*>(codes),
                           exponents, block_ids, num_block_ids, static_cast<uint4*>(out),
                           static_cast<uint32_t>(shape->num_kv_heads),
                           static_cast<uint32_t>(shape->head_dim / 16),
                           static_cast<uint32_t>(shape->block_size), shape->num_blocks);
    };
    if (dtype == SCA_DTYPE_F16) {
        launch(sca_hip::kv8_gather_kernel<sca_hip::F16>);
    } else {
        launch(sca_hip::kv8_gather_kernel<sca_hip::BF16>);
    }
    return sca_hip::CheckLaunch("kv8_gather_kernel", s);
}

}  // extern "C"
